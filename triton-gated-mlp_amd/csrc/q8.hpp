// 8-bit integer weights and activations: what the kernels of q8.hip and q8_gemm.hip and the C entry points share.
//
//   row of numbers v -> n = 127 v / max|v| rounded half to even, scale = max|v| / 127
//   y[t, c] = s_t s_c sum_r n_tr n_cr (+ bias)            sums of integers, exact in 32 bits
//
// Token rows and weights lie in the same order: tiles of 16 rows, and in a tile blocks of 64 integers of each row,
// [quarter of the 64][row][16], 1 KiB, a fragment of v_mfma_i32_16x16x64_i8 as a wavefront's lanes load it.  Columns are padded
// with zeros to multiples of 128.
#pragma once
#include "common.hpp"

namespace gmlp {

constexpr int Q8_MAX_COLS = 131072;   // 127 * 127 * 131072 < 2^31
constexpr int Q8_FEW_ROWS = 128;      // token rows that the weight-streaming kernels take at most
inline __host__ __device__ int64_t q8_padded(int64_t cols) { return (cols + 127) / 128 * 128; }
inline __host__ __device__ int64_t q8_tiled_rows(int64_t rows) { return (rows + 15) / 16 * 16; }

// Some rows of one expert: what a workgroup takes at a time.  `row`: of the first in the rows' own order, a multiple of 16.
struct Q8Tile {
  int expert, row, rows, unused;
};
// The choices of a call in the order of their experts; device pointers into the caller's workspace.  An expert's rows begin at a
// multiple of 16.
struct Q8Plan {
  int* total;        // [3] tiles in `tiles`, rows with those left empty between experts, tiles in `large`
  Q8Tile* tiles;     // in ascending order of expert and row
  Q8Tile* large;     // the same rows in tiles of 256 (nullable)
  int* row_of;       // [M * top_k]: row of a choice, -1 where its expert is not run
  int* token_of;     // [rows]: -1 where a row is left empty
};
// Token rows as integers one behind the other, [rows][padded], for the experts' workgroups to find by their numbers: each once, and
// without the plan.
struct Q8Lines {
  const void* x;  // [rows][cols]
  int8_t* codes;
  float* scales;
  int rows, cols, padded, dtype;
};
constexpr int64_t Q8_MAX_LINES = 0x7ffe0000;  // bytes: what offsets of 31 bits and a row reach
inline int64_t q8_plan_rows(int64_t pairs, int64_t E) {  // at most
  const int64_t most = E + pairs / 16;
  return 16 * (pairs < most ? pairs : most);
}
inline int64_t q8_plan_tiles(int64_t pairs, int64_t E, int64_t cap) { return pairs / cap + (pairs < E ? pairs : E); }

// One product, dense (tiles = NULL: `M` rows, one matrix) or of the rows and experts of a plan, with a stage's epilogue:
//   SETS = 2   out[m, n] = act(gate + b_gate) * (up + b_up) in T
//   SETS = 1   out[m, n] = product + bias in T, or (out_f32) product in float
struct Q8Product {
  const int8_t* x;       // [rows / 16][K / 64][1024]
  const float* sx;       // [rows]
  const int8_t* w[2];    // [experts][N / 16][K / 64][1024]
  const float* sw[2];    // [experts][N]
  const void* bias[2];   // [N], nullable
  void* out;             // [rows][N]
  int M, N, K, act;      // K: padded
  int out_f32;
  const Q8Tile* tiles;
  const int* total;      // how many tiles there are
  int most_tiles;        // ... at most
  const int* token_of;   // streaming, SETS = 2 or launch_q8_few_rows: the tiles' rows are those of these tokens (nullable: their own);
  int tokens;            // ... launch_q8_few: x and sx are Q8Lines of so many
  int most_rows;         // launch_q8_few_rows: rows of a tile, at most
  int nxcd, cus;
  // GEMM only
  int tile_class, splits, rotate, group_m;
  int first_col, cols;   // the output columns of this launch (all of them where splits > 1)
  float* partial;        // [splits][SETS][M][N] 32-bit sums, where splits > 1 (dense only)
};

// Weight streaming: the rows of a tile are at most 16 * token_tiles (1, 2, 4 or 8).
template <typename T>
hipError_t launch_q8_few(const Q8Product& p, int sets, int token_tiles, hipStream_t s);
// An expert layer's only token: its logits, and where its choices are left.
constexpr int Q8_SOLO_MAX_E = 256;
struct Q8Solo {
  const void* logits;  // [E] of a GMLP_* type
  int logits_dtype, E, top_k, normalize;
  int* experts;        // [top_k], < 0: not run
  float* weights;      // [top_k]
};
// The same of rows [..][cols] as they are, p.most_rows in a tile, where q8_own_rows allows it (p.x and p.sx are not used): dense, of a
// plan's tiles, or (solo) the only token through the matrices of each of its choices, out [top_k][N].
bool q8_own_rows(int64_t most_rows, int64_t padded, int64_t N, int cus);
template <typename T>
hipError_t launch_q8_few_rows(const Q8Product& p, const T* rows, int cols, int sets, const Q8Solo* solo, hipStream_t s);
// y[N] = sum over the choices of weight * down(h), h [top_k][cols].  Where q8_solo says so.
bool q8_solo(int64_t M, int64_t E, int64_t top_k, int64_t padded_k, int64_t padded_n);
template <typename T>
hipError_t launch_q8_solo_down(const Q8Solo& solo, const T* h, const int8_t* w, const float* sw, T* y, int N, int cols, hipStream_t s);
// GEMM: tile_class LARGE (256 rows), WIDE or MEDIUM_FULL (128).
template <typename T>
hipError_t launch_q8_gemm(const Q8Product& p, int sets, hipStream_t s);

// Rows to integers: `count` matrices of `rows` rows (token_of: row r of the result is row token_of[r] of x, or none at -1; up
// to rows_at[0] rows), each padded to whole tiles.
template <typename T>
hipError_t launch_q8_rows(const T* x, int8_t* codes, float* scales, int64_t count, int64_t rows, int64_t cols, const int* token_of,
                          const int* rows_at, hipStream_t s);
template <typename T>
hipError_t launch_q8_dequantize(const int8_t* codes, const float* scales, T* w, int64_t count, int64_t rows, int64_t cols, hipStream_t s);
// The plan of routed choices; cap: rows of a tile.  A choice of weight 0 is not run.
// lines (nullable): what the launch's other workgroups do meanwhile; with it token_of is not -1 but left where no row is.
hipError_t launch_q8_plan(const int64_t* experts, const float* weights, const Q8Plan& plan, int M, int E, int top_k, int cap,
                          const Q8Lines* lines, hipStream_t s);
// Routing and plan of up to Q8_ROUTE_ROWS tokens from the logits on.  (8 of 64 experts, 64 tokens: 7.0 us, in two launches 4.7 and 4.7; for
// 256 tokens 15.8, 5 and 6.)
constexpr int Q8_ROUTE_ROWS = 128;
template <typename L>
hipError_t launch_q8_route_plan(const L* logits, float* weights, const Q8Plan& plan, int M, int E, int top_k, int normalize, int cap,
                                const Q8Lines* lines, hipStream_t s);
// y[t] = sum over the choices of weight * parts[row]
template <typename T>
hipError_t launch_q8_combine(const float* parts, const float* weights, const int* row_of, T* y, int64_t M, int64_t K, int top_k,
                             hipStream_t s);

}  // namespace gmlp
