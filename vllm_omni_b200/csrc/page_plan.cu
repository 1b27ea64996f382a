// Pages and slots of one step, planned on the GPU from the sequences' lengths, and pages given back.
//
//   omni_plan_step      prefix sums over the new tokens and over the pages they need; pages from the top of the stack of free ones, in the order of the
//                       sequences; block table entries, slots, positions, sequence and visible keys of every row of the batch
//   omni_release_pages  the pages of finished sequences back onto the stack
//
// A step moves 24 bytes a row, so a call is a launch and the latency of two dependent scans.  One cluster does it all: every block repeats the scans over
// at most 4096 sequences in its own shared memory (less than a barrier across the grid would take) and then writes its share of the rows, each of which
// finds its sequence by bisection of the starts.  The lengths and the stack's height may be written in place: a barrier of the cluster lies between the
// blocks' reads and the first block's writes.  One sequence and row 5.3 us, where a launch that does nothing takes 2.4; 256 6.3; 12289 rows 8.2; 4096 sequences of four
// rows 10.6, released 12.
#include "host_util.h"
#include "ptx_sm100.cuh"

namespace omni {

constexpr int PP_THREADS = 1024, PP_MAX_SEQS = 4096, PP_PER = PP_MAX_SEQS / PP_THREADS;

struct PlanStep {
  const int *context, *fresh;            // [S] cached tokens, new tokens
  int* tables;                           // [S, W] at table_stride
  const int *free_pages, *n_free;        // the stack, its height
  int *q_start, *lens, *slots;           // [S + 1], [S], [rows]
  long long* positions;                  // [rows]
  int *row_seq, *row_lens, *n_free_out;  // [rows], [rows], [1]
  int *context_io, *n_free_io;           // advance: the same lengths and height once more, in place; else null
  int* status;
  long table_stride;
  int S, W, page, rows, pages, capacity; // ids lie below `pages`; entries of the stack
};

// Pages that n tokens fill
__device__ __forceinline__ int pages_of(int n, int page) { return n > 0 ? (n - 1) / page + 1 : 0; }

// Exclusive prefix sums of PP_PER consecutive values per thread; the block's total in `total`.
__device__ __forceinline__ void block_scan(long long (&v)[PP_PER], long long& total, long long* sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long mine = 0;
#pragma unroll
  for (int i = 0; i < PP_PER; ++i) {
    const long long x = v[i];
    v[i] = mine;
    mine += x;
  }
  long long run = mine;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const long long up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  __syncthreads();                       // the previous use of `sh` is over
  if (lane == 31) sh[warp] = run;
  __syncthreads();
  if (warp == 0) {
    long long w = sh[lane];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const long long up = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += up;
    }
    sh[lane] = w;
  }
  __syncthreads();
  total = sh[31];
  const long long before = run - mine + (warp ? sh[warp - 1] : 0);
#pragma unroll
  for (int i = 0; i < PP_PER; ++i) v[i] += before;
}

__global__ void __launch_bounds__(PP_THREADS)
plan_step_kernel(const __grid_constant__ PlanStep p) {
  extern __shared__ int sm[];
  __shared__ long long sh[32];
  const int S = p.S;
  int *start = sm, *ctx = sm + S + 1, *taken = ctx + S, *base = taken + S;
  const uint32_t rank = cluster_ctarank();
  pdl_begin();
  const int height = min(max(0, *p.n_free), p.capacity);
  const long long most = (long long)p.W * p.page;

  long long v[PP_PER];
  int c[PP_PER], n[PP_PER], mine[PP_PER];
  const int s0 = threadIdx.x * PP_PER;
#pragma unroll
  for (int i = 0; i < PP_PER; ++i) {
    const bool in = s0 + i < S;
    c[i] = in ? (int)min((long long)max(p.context[s0 + i], 0), most) : 0;
    v[i] = n[i] = in ? min(max(p.fresh[s0 + i], 0), p.rows) : 0;
  }
  long long total;
  block_scan(v, total, sh);
  const int live = (int)min(total, (long long)p.rows);
#pragma unroll
  for (int i = 0; i < PP_PER; ++i) {
    const int at = (int)min(v[i], (long long)p.rows);
    if (s0 + i < S) {
      start[s0 + i] = at;
      ctx[s0 + i] = c[i];
    }
    n[i] = min(n[i], p.rows - at);
    mine[i] = pages_of(c[i], p.page);
    v[i] = max(0LL, min((long long)p.W, ((long long)c[i] + n[i] + p.page - 1) / p.page) - mine[i]);
  }
  if (threadIdx.x == 0) start[S] = live;
  int need[PP_PER];
#pragma unroll
  for (int i = 0; i < PP_PER; ++i) need[i] = (int)v[i];
  block_scan(v, total, sh);
#pragma unroll
  for (int i = 0; i < PP_PER; ++i) {
    const int got = (int)min((long long)need[i], max(0LL, height - v[i]));
    const long long room = ((long long)mine[i] + got) * p.page - c[i];
    n[i] = (int)min((long long)n[i], max(room, 0LL));
    if (s0 + i < S) {
      taken[s0 + i] = n[i];
      base[s0 + i] = (int)min(v[i], (long long)height);
    }
  }
  if (gridDim.x > 1) cluster_sync_all(); // the shared arrays are written, and every block has read the lengths and the height
  else __syncthreads();
  if (rank == 0) {
    const int left = height - (int)min(total, (long long)height);
    for (int s = threadIdx.x; s <= S; s += PP_THREADS) p.q_start[s] = start[s];
    for (int s = threadIdx.x; s < S; s += PP_THREADS) {
      const int l = ctx[s] + taken[s];
      p.lens[s] = l;
      if (p.context_io) p.context_io[s] = l;
    }
    if (threadIdx.x == 0) {
      *p.n_free_out = left;
      if (p.n_free_io) *p.n_free_io = left;
    }
  }
  const long stride = (long)gridDim.x * PP_THREADS;
  for (long t = (long)blockIdx.x * PP_THREADS + threadIdx.x; t < p.rows; t += stride) {
    int slot = -1, seq = -1, keys = 0;
    long long pos = 0;
    if (t < live) {
      int lo = 0, hi = S;                // the last sequence that starts at or before t: later ones that start there have no rows before the next start
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= t) lo = mid; else hi = mid;
      }
      seq = lo;
      const int i = (int)t - start[seq], first = pages_of(ctx[seq], p.page);
      pos = (long long)ctx[seq] + i;
      if (i < taken[seq]) {
        const int col = (int)(pos / p.page), off = (int)(pos - (long long)col * p.page);
        int* entry = p.tables + (long)seq * p.table_stride + col;
        const int page = col < first ? *entry : p.free_pages[height - 1 - base[seq] - (col - first)];
        if (page >= 0 && page < p.pages) {
          slot = page * p.page + off;
          keys = (int)pos + 1;
        } else {
          atomicCAS(p.status, 0, ERR_BOUNDS);
        }
        if (col >= first && off == 0) *entry = page;       // a new page's first token is always among those taken
      }
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
    p.row_seq[t] = seq;
    p.row_lens[t] = keys;
  }
}

struct ReleasePages {
  int* lens;                             // [S]; 0 afterwards where done
  const unsigned char* done;             // [S]
  const int* tables;
  int *free_pages, *n_free, *status;
  long table_stride;
  int S, W, page, pages, capacity;       // ids lie below `pages`; entries of free_pages
};

__global__ void __launch_bounds__(PP_THREADS)
release_pages_kernel(const __grid_constant__ ReleasePages p) {
  extern __shared__ int sm[];
  __shared__ long long sh[32];
  __shared__ int bad, fits;
  int *at = sm, *count = sm + p.S;
  if (threadIdx.x == 0) bad = fits = 0;
  pdl_begin();
  const int height = min(max(0, *p.n_free), p.capacity);
  long long v[PP_PER], total;
  int n[PP_PER];                         // pages of a sequence that is done, else -1
  const int s0 = threadIdx.x * PP_PER;
#pragma unroll
  for (int i = 0; i < PP_PER; ++i) {
    const int s = s0 + i;
    const bool done = s < p.S && p.done[s];
    v[i] = done ? min(p.W, pages_of(p.lens[s], p.page)) : 0;
    n[i] = done ? (int)v[i] : -1;
  }
  block_scan(v, total, sh);
  const int room = p.capacity - height;
  int end = 0;                           // of the thread's last sequence that fits
#pragma unroll
  for (int i = 0; i < PP_PER; ++i) {
    const int s = s0 + i;
    const bool whole = n[i] <= 0 || v[i] + n[i] <= room;  // else it keeps its pages and its length, and so do those behind it
    if (s < p.S) {
      at[s] = (int)min(v[i], (long long)room);
      count[s] = whole ? max(n[i], 0) : 0;
      if (n[i] >= 0 && whole) p.lens[s] = 0;
      if (count[s]) end = at[s] + n[i];
    }
  }
  end = __reduce_max_sync(0xffffffffu, end);
  if ((threadIdx.x & 31) == 0 && end) atomicMax(&fits, end);
  __syncthreads();                       // every thread has read the height
  const int back = fits;
  if (threadIdx.x == 0) {
    *p.n_free = height + back;
    if (total > room) atomicCAS(p.status, 0, ERR_BOUNDS);
  }
  const int lane = threadIdx.x & 31;
  int* stack = p.free_pages + height;
  bool odd = false;
  for (int s = threadIdx.x >> 5; s < p.S; s += PP_THREADS / 32)
    for (int i = lane; i < count[s]; i += 32) {
      const int id = p.tables[(long)s * p.table_stride + i];
      odd |= id < 0 || id >= p.pages;
      stack[at[s] + i] = id;
    }
  if (odd) bad = 1;
  __syncthreads();
  if (!bad || threadIdx.x >= 32) return;
  // Ids that no page has are reported, and the others move up: no entry is written before it has been read.
  int to = 0;
  for (int i0 = 0; i0 < back; i0 += 32) {
    const int id = i0 + lane < back ? stack[i0 + lane] : -1;
    const bool ok = id >= 0 && id < p.pages;
    const unsigned m = __ballot_sync(0xffffffffu, ok);
    if (ok) stack[to + __popc(m & ((1u << lane) - 1))] = id;
    to += __popc(m);
    __syncwarp();
  }
  if (lane == 0) {
    *p.n_free = height + to;
    atomicCAS(p.status, 0, ERR_BOUNDS);
  }
}

}  // namespace omni

using namespace omni;

// Shapes as in PlanStep; context_io / n_free_io may be null or the operands themselves.  At most 4096 sequences.
extern "C" int omni_plan_step(const int* context, const int* fresh, int* tables, long table_stride, const int* free_pages, const int* n_free, int S, int W,
                              int page, int rows, int pages, int capacity, int* q_start, int* lens, int* slots, long long* positions, int* row_seq, int* row_lens,
                              int* n_free_out, int* context_io, int* n_free_io, int* status, void* stream) {
  if (S < 0 || S > PP_MAX_SEQS || W < 1 || page < 1 || rows < 0 || pages < 1 || capacity < 0 || (long)pages * page > 0x7fffffffL || (long)W * page > 0x7fffffffL) return RC_BAD_ARG;
  PlanStep p = {context, fresh, tables, free_pages, n_free, q_start, lens, slots, positions, row_seq, row_lens, n_free_out, context_io, n_free_io, status,
                table_stride, S, W, page, rows, pages, capacity};
  // one block while its threads have at most two rows each, else eight
  const int blocks = rows <= 2 * PP_THREADS ? 1 : 8;
  const int smem = (4 * S + 1) * 4;
  static unsigned long long ready = 0;
  if (smem > 47 * 1024)
    if (int e = ensure_dynamic_smem((const void*)plan_step_kernel, (4 * PP_MAX_SEQS + 1) * 4, ready)) return e;
  launch_with(true, blocks, plan_step_kernel, blocks, PP_THREADS, smem, (cudaStream_t)stream, p);
  return (int)cudaGetLastError();
}

extern "C" int omni_release_pages(int* lens, const unsigned char* done, const int* tables, long table_stride, int* free_pages, int* n_free, int S, int W, int page,
                                  int pages, int capacity, int* status, void* stream) {
  if (S <= 0) return RC_OK;
  if (S > PP_MAX_SEQS || W < 1 || page < 1 || pages < 1 || capacity < 0) return RC_BAD_ARG;
  ReleasePages p = {lens, done, tables, free_pages, n_free, status, table_stride, S, W, page, pages, capacity};
  launch_overlapped(release_pages_kernel, 1, PP_THREADS, 2 * S * 4, (cudaStream_t)stream, p);
  return (int)cudaGetLastError();
}
