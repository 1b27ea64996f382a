// Low-bit rows and their products: entry points.
//
//  omni_lowbit_rows        rows of bf16 -> codes and scales; optionally the residual's addition and the RMS norm before it   (lowbit_rows.cuh)
//  omni_lowbit_dequantize  codes and scales -> bf16 or fp32
//  omni_lowbit_linear      linear layer on a packed weight: rows as bf16 (quantised first, in the caller's workspace) or quantised  (fp4_gemm.cuh)
//  omni_lowbit_experts     both products of a mixture of experts, by the tables of a plan (moe.cu)
#include "fp4_gemm.cuh"
#include "lowbit_rows.cuh"

using namespace omni;

// gain null: x is quantised as it is.  Else s = x + residual (rounded to bf16, stored in total where given), rows s / rms(s) * gain (bf16, stored in
// normed where given) are.  group: rows of a weight's matrix (rows, for one).
extern "C" int omni_lowbit_rows(const void* x, long ldx, long rows, int K, long group, int fmt, const void* residual, long ldr, const void* gain,
                                float eps, void* total, long ldt, void* normed, long ldn, void* codes, void* scales, void* row_scale,
                                void* stream) {
  RowsArgs a = {};
  a.x = (const bf16*)x; a.residual = (const bf16*)residual; a.gain = (const bf16*)gain; a.total = (bf16*)total; a.normed = (bf16*)normed;
  a.ldx = ldx; a.ldr = ldr; a.ldt = ldt; a.ldn = ldn; a.rows = rows; a.K = K; a.eps = eps;
  a.codes = (uint8_t*)codes; a.scales = scales; a.row_scale = (float*)row_scale;
  a.place.group = group > 0 ? group : 1;
  return rows_any(a, fmt, (cudaStream_t)stream);
}

extern "C" int omni_lowbit_dequantize(const void* codes, const void* scales, const void* row_scale, long rows, int K, long group, int fmt,
                                      int f32, void* out, void* stream) {
  return dequantize_any({(const uint8_t*)codes, scales, (const float*)row_scale, out, rows, group > 0 ? group : 1, K, f32}, fmt, (cudaStream_t)stream);
}

// y [M, N] (gated: [M, N / 2]) of x [M, K] and w [N, K].  raw (bf16 rows, pitch ldx) not null: quantised into x, xs, xf first.  force_tile 0: by the rules
// of fp4_gemm.cuh, 16 / 64 / 128 / 256; force_split 0: by the rules, 1 / 2 / 4 / 8.
extern "C" int omni_lowbit_linear(const void* raw, long ldx, void* x, void* xs, void* xf, const void* w, const void* ws, const void* wf, void* y, long ldy,
                                  long M, int N, int K, int fmt, int gated, const void* bias, int act, const void* gate, long gate_stride,
                                  long rows_per_gate, const void* residual, long ldr, int force_tile, int force_split, void* status, void* stream) {
  if (M <= 0 || N <= 0 || K <= 0) return RC_OK;
  if (M > 0x7fffff00L || K % 32 || (gated && (N % 16 || bias || act || gate || residual)) || act < 0 || act > 2) return RC_BAD_ARG;
  if (gate && rows_per_gate < 1) return RC_BAD_ARG;
  Fp4Args a = {};
  a.y = (bf16*)y; a.ldy = ldy; a.wf = (const float*)wf; a.xf = (const float*)xf;
  a.bias = (const bf16*)bias; a.residual = (const bf16*)residual; a.gate = (const bf16*)gate;
  a.ldr = ldr; a.gate_stride = gate_stride; a.rows_per_gate = (int)rows_per_gate; a.act = act;
  a.M = (int)M; a.N = N; a.K = K;
  a.by16 = N % 8 == 0 && ldy % 8 == 0 && ldr % 8 == 0 && gate_stride % 8 == 0 && on16(y) && on16(bias) && on16(gate) && on16(residual);
  const int rc = pick_tiles(a, force_tile, force_split);
  if (rc < 0) return rc;
  if (raw) {
    if (int e = omni_lowbit_rows(raw, ldx, M, K, M, fmt, nullptr, 0, nullptr, 0.f, nullptr, 0, nullptr, 0, x, xs, xf, stream)) return e;
  }
  return launch_any(a, {w, ws, x, xs, 1, M, (M + 127) / 128}, fmt, gated != 0, rc, (int*)status, (cudaStream_t)stream);
}

struct ExpertOperand {           // one product's rows in a workspace, and its weights
  void *codes, *scales, *row_scale;
  const void *w, *ws, *wf;
  int N, K;
};

// Rows of x (pair p reads row p / per, pairs a multiple of per) through `up` (gated, N = 2 F) to h [pairs, F] and through `down` to y [pairs, D], both in the plan's order of rows;
// tile: the most rows a tile has, 64 / 128 / 256; n_rows: how many rows the
// plan has; place_of_row [pairs]: scratch.
extern "C" int omni_lowbit_experts(const void* x, long ldx, int per, long pairs, int experts, int fmt, const ExpertOperand* up, const ExpertOperand* down, void* h,
                                   void* y, const int* row_of_pair, const int* tile_expert, const int* tile_row0, const int* tile_rows, int max_tiles,
                                   int tile, const int* n_rows, int* place_of_row, void* status, void* stream) {
  if (pairs <= 0 || max_tiles <= 0) return RC_OK;
  if (pairs > 0x7fffff00L || per < 1 || experts < 1 || !row_of_pair || !n_rows || !place_of_row || pairs % per || !tile_expert || !tile_row0 || !tile_rows || up->N % 16 || up->N != 2 * down->K ||
      up->K % 32 || down->K % 32 || fmt == FMT_FP8)
    return RC_BAD_ARG;
  cudaStream_t s = (cudaStream_t)stream;
  const int pitch = tile > 128 ? 256 : 128;
  for (int half = 0; half < 2; ++half) {
    const ExpertOperand& o = half ? *down : *up;
    RowsArgs r = {};
    r.x = (const bf16*)(half ? h : x); r.ldx = half ? o.K : ldx; r.rows = half ? pairs : pairs / per; r.K = o.K;
    r.codes = (uint8_t*)o.codes; r.scales = o.scales; r.row_scale = (float*)o.row_scale;
    r.place = {1, half ? nullptr : row_of_pair, tile_expert, tile_row0, tile_rows, n_rows, place_of_row, per, max_tiles, pitch};
    if (int e = rows_any(r, fmt, s)) return e;
    Fp4Args a = {};
    a.y = (bf16*)(half ? y : h); a.ldy = half ? o.N : o.N / 2; a.wf = (const float*)o.wf; a.xf = (const float*)o.row_scale;
    a.M = (int)pairs; a.N = o.N; a.K = o.K; a.rows_per_gate = 1; a.split = 1;
    a.by16 = a.N % 8 == 0 && a.ldy % 8 == 0 && on16(a.y);
    a.tile_expert = tile_expert; a.tile_row0 = tile_row0; a.tile_rows = tile_rows; a.max_tiles = max_tiles;
    if (int e = launch_any(a, {o.w, o.ws, o.codes, o.scales, experts, pairs, (long)max_tiles * (pitch / 128)}, fmt, half == 0, tile, (int*)status, s)) return e;
  }
  return RC_OK;
}
