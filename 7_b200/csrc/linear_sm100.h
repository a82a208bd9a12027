// Internal interface between the C-ABI backend and the sm_100a kernels of the
// linear layers: matrix products with bias, activation and residual in their
// epilogue, dense or grouped by expert, and the products of their backward pass.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace wave {

enum LinearAct : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };

// Which extent of a product follows the experts' offsets.
enum LinearRagged : int {
  kRaggedNone = 0,
  kRaggedRows = 1, // the token rows of the output (forward, input gradient)
  kRaggedK = 2,    // the contraction (weight gradient): one output matrix for each expert
};

constexpr int kLinearMaxGroups = 1024; // two ints of shared memory for each
constexpr int kLinearMaxSplits = 8;    // CTAs of a cluster that share one tile's contraction

// Kernel-space product D[P x Q] = A[P x K] * B[Q x K]^T.  The P side takes the
// 128 rows of the tensor core's tile, the Q side its 16..256 columns.  With
// `swap` the features are on the P side and the tokens on the Q side (few
// tokens), otherwise tokens are rows; the weight gradient has out-features on P
// and in-features on Q.  D's element (token m, feature n) is at m * ldd + n
// either way.
struct FastDiv { // see fast_div
  uint32_t d, m, s;
};
inline FastDiv make_fast_div(uint32_t d) {
  FastDiv f{d, 0, 0};
  while ((1ull << f.s) < d)
    ++f.s;
  if (f.s > 0)
    f.m = static_cast<uint32_t>(((1ull << (31 + f.s)) + d - 1) / d);
  return f;
}

struct LinearParams {
  int P, Q, K;       // extents; the ragged one is its upper bound (all tokens)
  int ragged, groups;
  const int *offsets; // [groups + 1], on the device; null when not ragged
  int group_a, group_b; // the operand has one matrix for each group (third coordinate of its tensor map)
  int chunks_a, chunks_b; // an MN-major operand's map is one over 64-column chunks: a stage of it is one copy
  int tile_q;        // columns of a tile <= the kernel's: a multiple of 16, of 64 where B is stored [K][Q]
  int p_blocks, q_blocks; // tiles along each side (ragged side: unused)
  int raster_log2;   // row blocks (its power of two) that are walked down before the next column block
  FastDiv band_tiles;  // tiles of so many row blocks
  FastDiv group_tiles; // weight gradient: tiles of a group
  int stages;        // ring depth of this launch (at most the kernel's)
  int splits;        // CTAs of a cluster that share a tile's contraction; then one tile for each cluster
  int is_bf16;       // operands, z, residual and 16-bit outputs: bf16 or f16
  int act;
  // D
  void *D;
  long long ldd, group_d;
  void *Z;           // pre-activation, 16-bit, or null
  long long ldz;
  const void *R;     // residual, 16-bit, or null
  long long ldr;
  const void *bias;  // or null
  int bias_f32;
  long long group_bias;
  int vec_d, vec_z, vec_r; // 16-byte accesses are aligned in D / Z / R
  int tma_d, tma_z;  // whole blocks of D / Z leave by TMA stores (tokens as rows, the maps are there)
  int zero_rest;     // rows of D and Z that belong to no group are set to zero
  int beside;        // runs beside the launch before it (see start_after_previous)
};

struct LinearLaunch {
  int a_mn, b_mn; // operand stored with the contraction as its slow direction
  int swap;
  int tile_n;     // kernel instantiation: 16, 32, 64, 128 or 256 columns
  int out_f32;
  int grid;       // CTAs (a multiple of splits)
  int pair;       // CTA-pair kernel: 256 x tile_q tiles, 16-bit results, tokens as rows or (with experts) columns
  int pdl;        // launch with programmatic stream serialization
};

// Bytes of the experts' table in shared memory.
constexpr int linear_table_bytes(int ragged, int groups) { return ragged == kRaggedNone ? 0 : 2 * 4 * (groups + 1); }
// Ring depth the kernel has room for beside it; a launch may take fewer stages, at least 3.
int linear_max_stages(int tile_n, int out_f32, int ragged, int groups);
int linear_pair_stages(int ragged, int groups); // (taken whole)
struct LinearMaps {
  CUtensorMap a, b, d, z; // d and z: read where tma_d / tma_z are set, boxes of 64 (forward, 16-bit) or 128 bytes x 32 rows
};
cudaError_t launch_linear(const LinearMaps &m, const LinearParams &p, const LinearLaunch &l, cudaStream_t stream);
cudaError_t linear_read_status(int out[4], bool clear);
// tile_q a multiple of 32 (of 128 where B is stored [K][Q]) up to 256; grid even.
// With swap (experts only) tile_q bounds the tokens of a tile.
cudaError_t launch_linear_pair(const LinearMaps &m, const LinearParams &p, const LinearLaunch &l, cudaStream_t stream);
cudaError_t linear_pair_read_status(int out[4], bool clear);

// ---- helpers around the products (linear_aux_sm100.cu)
// 16-bit rows with any stride into rows of `ld_dst` elements: what a TMA load
// needs (16-byte strides) of an operand that does not have it.  groups = 0: nothing.
struct PackRows {
  const void *src;
  long long ld_src, group_src;
  void *dst;
  long long ld_dst, group_dst;
  int rows, cols, groups;
  const int *offsets; // not null: matrices of groups without any of the `tokens` rows are neither read nor written
  int tokens;
};
// x is one matrix, the weights one or one for each group; either may be nothing.
cudaError_t launch_pack_rows(const PackRows &x, const PackRows &weights, int pdl, cudaStream_t stream);

// dz = dy * act'(z), rounded to the operands' type, and the column sums of the
// unrounded dz (dbias) of each group in two steps of fixed order.
struct LinearActGrad {
  int rows, cols, groups;
  const int *offsets; // null: one group of all rows
  int act, is_bf16, dy_f32;
  const void *dY;
  long long ldy;
  const void *Z; // null when act is none
  long long ldz;
  void *dZ; // null: column sums only
  long long lddz;
  float *partial; // [chunks][cols] (short groups: [blocks][cols], unused where one launch does it), null: no column sums
  int chunk_rows;
  void *dbias; // [groups][cols]
  int dbias_type; // 0 f32, 1 f16, 2 bf16
  int vec_dy, vec_z;
  int short_groups; // all rows of a group to a block, up to a limit
  int short_cols;   // columns of such a block, 32 or 64
  int pdl;
};
int linear_act_grad_chunks(int rows, int groups, int chunk_rows); // upper bound, sizes `partial`
// Short groups (groups = 0: one of all rows): how many blocks there can be beside one for each group.  None: no group can
// exceed a block, and one launch without `partial` does it all.
int linear_act_grad_short_more(int rows, int groups);
cudaError_t launch_act_grad(const LinearActGrad &p, cudaStream_t stream);
cudaError_t launch_column_sums(const LinearActGrad &p, cudaStream_t stream); // what act_grad leaves of dbias

} // namespace wave
