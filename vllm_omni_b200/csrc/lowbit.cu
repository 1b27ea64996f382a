// Low-bit rows and their products: entry points.
//
//  omni_lowbit_rows        rows of bf16 -> codes and scales; optionally the residual's addition and the RMS norm before it   (lowbit_rows.cuh)
//  omni_lowbit_dequantize  codes and scales -> bf16 or fp32
//  omni_lowbit_linear      linear layer on a packed weight: rows as bf16 (quantised first, in the caller's workspace) or quantised  (fp4_gemm.cuh)
//  omni_lowbit_experts     both products of a mixture of experts, by the tables of a plan (moe.cu)
//
// Each takes its operands as one block of 8-byte fields: a layer's 26 passed one by one cost a Python caller 3 us, of 6 for the whole call.
#include "fp4_gemm.cuh"
#include "lowbit_rows.cuh"

using namespace omni;

// gain null: x is quantised as it is.  Else s = x + residual (rounded to bf16, stored in total where given), rows s / rms(s) * gain (bf16, stored in
// normed where given) are.  group: rows of a weight's matrix (rows, for one).
struct LowbitRows {
  const void* x;
  long ldx, rows, K, group, fmt;
  const void* residual;
  long ldr;
  const void* gain;
  double eps;
  void* total;
  long ldt;
  void* normed;
  long ldn;
  void *codes, *scales, *row_scale, *stream;
};
extern "C" int omni_lowbit_rows(const LowbitRows* c) {
  RowsArgs a = {};
  a.x = (const bf16*)c->x; a.residual = (const bf16*)c->residual; a.gain = (const bf16*)c->gain; a.total = (bf16*)c->total; a.normed = (bf16*)c->normed;
  a.ldx = c->ldx; a.ldr = c->ldr; a.ldt = c->ldt; a.ldn = c->ldn; a.rows = c->rows; a.K = (int)c->K; a.eps = (float)c->eps;
  a.codes = (uint8_t*)c->codes; a.scales = c->scales; a.row_scale = (float*)c->row_scale;
  a.place.group = c->group > 0 ? c->group : 1;
  return rows_any(a, (int)c->fmt, (cudaStream_t)c->stream);
}

struct LowbitValues {
  const void *codes, *scales, *row_scale;
  long rows, K, group, fmt, f32;
  void *out, *stream;
};
extern "C" int omni_lowbit_dequantize(const LowbitValues* c) {
  return dequantize_any({(const uint8_t*)c->codes, c->scales, (const float*)c->row_scale, c->out, c->rows, c->group > 0 ? c->group : 1, (int)c->K, (int)c->f32},
                        (int)c->fmt, (cudaStream_t)c->stream);
}

// y [M, N] (gated: [M, N / 2]) of x [M, K] and w [N, K].  raw (bf16 rows, pitch ldx) not null: quantised into x, xs, xf first.  force_tile 0: by the rules
// of fp4_gemm.cuh, 16 / 64 / 128 / 256; force_split 0: by the rules, 1 / 2 / 4 (256: 1 / 2).
struct LowbitLinear {
  const void* raw;
  long ldx;
  void *x, *xs, *xf;
  const void *w, *ws, *wf;
  void* y;
  long ldy, M, N, K, fmt, gated;
  const void* bias;
  long act;
  const void* gate;
  long gate_stride, rows_per_gate;
  const void* residual;
  long ldr, force_tile, force_split;
  void *status, *stream;
};
extern "C" int omni_lowbit_linear(const LowbitLinear* c) {
  if (c->M <= 0 || c->N <= 0 || c->K <= 0) return RC_OK;
  if (c->M > 0x7fffff00L || c->N > 0x7fffff00L || c->K > 0x7fffff00L || c->K % 32 || c->act < 0 || c->act > 2 || (c->gate && c->rows_per_gate < 1) ||
      (c->gated && (c->N % 16 || c->bias || c->act || c->gate || c->residual)))
    return RC_BAD_ARG;
  Fp4Args a = {};
  a.y = (bf16*)c->y; a.ldy = c->ldy; a.wf = (const float*)c->wf; a.xf = (const float*)c->xf;
  a.bias = (const bf16*)c->bias; a.residual = (const bf16*)c->residual; a.gate = (const bf16*)c->gate;
  a.ldr = c->ldr; a.gate_stride = c->gate_stride; a.rows_per_gate = c->gate ? (int)c->rows_per_gate : 1; a.act = (int)c->act;
  a.M = (int)c->M; a.N = (int)c->N; a.K = (int)c->K;
  a.by16 = a.N % 8 == 0 && a.ldy % 8 == 0 && a.ldr % 8 == 0 && a.gate_stride % 8 == 0 && on16(a.y) && on16(a.bias) && on16(a.gate) && on16(a.residual);
  const int tile = pick_tiles(a, (int)c->force_tile, (int)c->force_split);
  if (tile < 0) return tile;
  if (c->raw) {
    RowsArgs r = {};
    r.x = (const bf16*)c->raw; r.ldx = c->ldx; r.rows = c->M; r.K = a.K;
    r.codes = (uint8_t*)c->x; r.scales = c->xs; r.row_scale = (float*)c->xf;
    r.place.group = c->M;
    if (int e = rows_any(r, (int)c->fmt, (cudaStream_t)c->stream)) return e;
  }
  return launch_any(a, {c->w, c->ws, c->x, c->xs, 1, c->M, (c->M + 127) / 128}, (int)c->fmt, c->gated != 0, tile, (int*)c->status, (cudaStream_t)c->stream);
}

// Rows of x (pair p reads row p / per, pairs a multiple of per) through `up` (gated, N = 2 F) to h [pairs, F] and through `down` to y [pairs, D], both in the
// plan's order of rows; tile: the most rows a tile has, 16 / 128 / 256; place_of_pair: for tiles from every 128 rows on (tile 256: 256); n_rows: how many rows the
// plan has; place_of_row [pairs]: scratch.
struct ExpertOperand {           // one product's rows in a workspace, and its weights
  void *codes, *scales, *row_scale;
  const void *w, *ws, *wf;
  long N, K;
};
struct LowbitExperts {
  const void* x;
  long ldx, per, pairs, experts, fmt;
  void *h, *y;
  const int *row_of_pair, *place_of_pair, *tile_expert, *tile_row0, *tile_rows;
  long max_tiles, tile;
  const int* n_rows;
  int* place_of_row;
  void *status, *stream;
  ExpertOperand up, down;
};
extern "C" int omni_lowbit_experts(const LowbitExperts* c) {
  const ExpertOperand &up = c->up, &down = c->down;
  if (c->pairs <= 0 || c->max_tiles <= 0) return RC_OK;
  if (c->pairs > 0x7fffff00L || c->per < 1 || c->pairs % c->per || c->experts < 1 || !c->row_of_pair || !c->place_of_pair || !c->n_rows || !c->place_of_row || !c->tile_expert ||
      !c->tile_row0 || !c->tile_rows || up.N % 16 || up.N != 2 * down.K || up.K != down.N || up.K % 32 || down.K % 32 || c->fmt == FMT_FP8)
    return RC_BAD_ARG;
  cudaStream_t s = (cudaStream_t)c->stream;
  const int pitch = c->tile > 128 ? 256 : 128;
  for (int half = 0; half < 2; ++half) {
    const ExpertOperand& o = half ? down : up;
    RowsArgs r = {};
    r.x = (const bf16*)(half ? c->h : c->x); r.ldx = half ? o.K : c->ldx; r.rows = half ? c->pairs : c->pairs / c->per; r.K = (int)o.K;
    r.codes = (uint8_t*)o.codes; r.scales = o.scales; r.row_scale = (float*)o.row_scale;
    r.place = {1, half ? nullptr : c->row_of_pair, c->place_of_pair, c->n_rows, c->place_of_row, (int)c->per};
    if (int e = rows_any(r, (int)c->fmt, s)) return e;
    Fp4Args a = {};
    a.y = (bf16*)(half ? c->y : c->h); a.ldy = half ? o.N : o.N / 2; a.wf = (const float*)o.wf; a.xf = (const float*)o.row_scale;
    a.M = (int)c->pairs; a.N = (int)o.N; a.K = (int)o.K; a.rows_per_gate = 1; a.split = 1;
    a.by16 = a.N % 8 == 0 && a.ldy % 8 == 0 && on16(a.y);
    a.tile_expert = c->tile_expert; a.tile_row0 = c->tile_row0; a.tile_rows = c->tile_rows; a.max_tiles = (int)c->max_tiles;
    if (int e = launch_any(a, {o.w, o.ws, o.codes, o.scales, (int)c->experts, c->pairs, c->max_tiles * (pitch / 128)}, (int)c->fmt, half == 0, (int)c->tile,
                           (int*)c->status, s))
      return e;
  }
  return RC_OK;
}
