// Host side of the linear layers (include/wave_cuda.h, "linear layers"): checks,
// workspace, tensor maps and the choice of tiles for the products with an
// epilogue, dense and grouped by expert, forward and backward.
#include "../../include/wave_cuda.h"
#include "backend_env.h"
#include "fa_sm100.h" // make_tensor_map_16bit
#include "linear_sm100.h"

#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <exception>

namespace wave { // wave_cuda_backend.cu
void set_last_error(const char *message);
int make_tensor_map_store(CUtensorMap *map, int type, void *base, const uint64_t *dims, const uint64_t *strides_bytes,
                          uint32_t row_bytes, uint32_t box_rows);
}

namespace {

using wave::LinearLaunch;
using wave::LinearParams;

int fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  wave::set_last_error(buf);
  return code;
}
int cuda_fail(cudaError_t err, const char *what) {
  return fail(WAVE_E_CUDA, "%s: %s", what, cudaGetErrorString(err));
}

// No C++ exception leaves a C entry (std::bad_alloc of the small host objects).
template <typename F> int guarded(F f) {
  try {
    return f();
  } catch (const std::exception &e) {
    return fail(WAVE_E_CUDA, "host side failed: %s", e.what());
  } catch (...) {
    return fail(WAVE_E_CUDA, "host side failed");
  }
}

int sm_count(int *out) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess)
    return cuda_fail(err, "cudaGetDevice");
  err = cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev);
  return err == cudaSuccess ? WAVE_OK : cuda_fail(err, "cudaDeviceGetAttribute");
}

long long round_up(long long v, long long a) { return (v + a - 1) / a * a; }
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ---------------------------------------------------------------- descriptor
// The descriptor with its zeros replaced by what they stand for.
struct Shape {
  wave_linear_desc d;
  bool grouped;
  int matrices; // weight matrices
};

Shape resolve(const wave_linear_desc &in) {
  Shape s;
  s.d = in;
  wave_linear_desc &d = s.d;
  s.grouped = d.experts > 0;
  s.matrices = s.grouped ? d.experts : 1;
  auto rows = [](long long &ld, int rows, long long cols) {
    // a single row has no stride: take one that every access likes
    if (ld == 0)
      ld = cols;
    if (rows <= 1)
      ld = round_up(cols, 8);
  };
  rows(d.ldx, d.tokens, d.in_features);
  rows(d.ldy, d.tokens, d.out_features);
  rows(d.ldr, d.tokens, d.out_features);
  rows(d.ldz, d.tokens, d.out_features);
  rows(d.lddx, d.tokens, d.in_features);
  rows(d.ldw, d.out_features, d.in_features);
  rows(d.lddw, d.out_features, d.in_features);
  // (one row to a matrix: the matrices follow one another without the padding
  // that `rows` assumed)
  if (d.expert_stride_w == 0)
    d.expert_stride_w = (in.ldw ? in.ldw : d.in_features) * static_cast<long long>(d.out_features);
  if (d.expert_stride_dw == 0)
    d.expert_stride_dw = (in.lddw ? in.lddw : d.in_features) * static_cast<long long>(d.out_features);
  return s;
}

int validate(const wave_linear_desc *d) {
  if (!d)
    return fail(WAVE_E_INVALID, "descriptor is null");
  if (d->tokens < 0)
    return fail(WAVE_E_INVALID, "tokens must be >= 0; got %d", d->tokens);
  if (d->tokens > 1 << 30 || d->out_features > 1 << 30 || d->in_features > 1 << 30)
    return fail(WAVE_E_INVALID, "tokens and features must be at most 2^30; got %d, %d and %d", d->tokens, d->out_features,
                d->in_features);
  if (d->out_features < 1 || d->in_features < 1)
    return fail(WAVE_E_INVALID, "out_features and in_features must be >= 1; got %d and %d", d->out_features,
                d->in_features);
  if (d->experts < 0 || d->experts > wave::kLinearMaxGroups)
    return fail(WAVE_E_INVALID, "experts must be between 0 (one weight matrix) and %d; got %d", wave::kLinearMaxGroups,
                d->experts);
  if (d->io_type != WAVE_BF16 && d->io_type != WAVE_F16)
    return fail(WAVE_E_UNSUPPORTED, "io_type must be bf16 or f16; got %d", d->io_type);
  const int types[4] = {d->y_type, d->bias_type, d->dweight_type, d->dbias_type};
  const char *names[4] = {"y_type", "bias_type", "dweight_type", "dbias_type"};
  for (int i = 0; i < 4; ++i)
    if (types[i] != d->io_type && types[i] != WAVE_F32)
      return fail(WAVE_E_UNSUPPORTED, "%s must be io_type or f32; got %d", names[i], types[i]);
  if (d->activation < WAVE_ACT_NONE || d->activation > WAVE_ACT_SILU)
    return fail(WAVE_E_INVALID, "activation must be one of none, relu, gelu, gelu_tanh, silu; got %d", d->activation);
  const long long lds[7] = {d->ldx, d->ldw, d->ldy, d->ldr, d->ldz, d->lddx, d->lddw};
  const char *ld_names[7] = {"ldx", "ldw", "ldy", "ldr", "ldz", "lddx", "lddw"};
  const int cols[7] = {d->in_features, d->in_features,  d->out_features, d->out_features,
                       d->out_features, d->in_features, d->in_features};
  for (int i = 0; i < 7; ++i)
    if (lds[i] != 0 && (lds[i] < cols[i] || lds[i] > (1ll << 36)))
      return fail(WAVE_E_INVALID, "%s must be 0 or between %d and 2^36 elements; got %lld", ld_names[i], cols[i], lds[i]);
  const Shape s = resolve(*d);
  if (s.grouped) {
    const long long strides[2] = {s.d.expert_stride_w, s.d.expert_stride_dw};
    const long long lds2[2] = {d->ldw ? d->ldw : d->in_features, d->lddw ? d->lddw : d->in_features};
    for (int i = 0; i < 2; ++i)
      if (strides[i] < lds2[i] * (d->out_features - 1) + d->in_features || strides[i] > (1ll << 38))
        return fail(WAVE_E_INVALID, "%s must be 0 or hold a whole matrix (at most 2^38 elements); got %lld",
                    i == 0 ? "expert_stride_w" : "expert_stride_dw", strides[i]);
  }
  // Tile counts stay far inside 32 bits: 16-token tiles of 128 features, 128 x 64 tiles of each gradient.
  const long long token_tiles = (static_cast<long long>(d->tokens) + 15) / 16 + s.matrices;
  const long long f_tiles = ((d->out_features > d->in_features ? d->out_features : d->in_features) + 63) / 64;
  const long long w_tiles = ((d->out_features + 127ll) / 128) * ((d->in_features + 63ll) / 64) * s.matrices;
  if (token_tiles * f_tiles > (1ll << 29) || w_tiles > (1ll << 29))
    return fail(WAVE_E_INVALID, "too many output tiles");
  return WAVE_OK;
}

// A 16-bit result is summed in one accumulator, whose truncation costs 1.2e-9 of the
// norm for each product (linear_sm100.cu), and its epilogue waits for the whole sum:
// 2^26 products, a million stages of up to 0.55 us where every SM reads DRAM, are half
// of the second after which a wait gives up.  f32 results are summed in pieces.
constexpr int kLongestSum16 = 1 << 26;
int check_sum(const char *result, int type, int products) {
  if (type == WAVE_F32 || products <= kLongestSum16)
    return WAVE_OK;
  return fail(WAVE_E_UNSUPPORTED, "%s in 16 bits takes sums of at most 2^26 products; got %d", result, products);
}

// ------------------------------------------------------------------ products
enum class Product { kForward, kInputGrad, kWeightGrad };

int ragged_of(Product kind, const Shape &s) {
  return !s.grouped ? wave::kRaggedNone : kind == Product::kWeightGrad ? wave::kRaggedK : wave::kRaggedRows;
}

// One 16-bit operand as the tensor maps see it: `rows` x `cols` of each matrix,
// cols contiguous.
struct Operand {
  const void *ptr;
  long long ld, group;
  int rows, cols, matrices;
  bool packed() const { return ld % 8 != 0 || (matrices > 1 && group % 8 != 0); }
  long long packed_ld() const { return round_up(cols, 8); }
  size_t packed_bytes() const {
    return packed() ? static_cast<size_t>(round_up(packed_ld() * 2 * rows * static_cast<long long>(matrices), 256)) : 0;
  }
};

// Describes the layout of an operand in `to` whose strides are not multiples of
// 16 bytes, and points it there; nothing for one that is fine as it is.  With
// `offsets` (the experts' weights) only of the experts that have rows.
wave::PackRows pack(Operand *o, char **to, const int *offsets = nullptr, int tokens = 0) {
  wave::PackRows p{};
  if (!o->packed())
    return p;
  const long long ld = o->packed_ld(), group = ld * o->rows;
  p = wave::PackRows{o->ptr, o->ld, o->matrices > 1 ? o->group : 0, *to, ld, group, o->rows, o->cols, o->matrices,
                     offsets, tokens};
  const size_t bytes = o->packed_bytes();
  o->ptr = *to;
  o->ld = ld;
  o->group = group;
  *to += bytes;
  return p;
}
int run_packs(const wave::PackRows &x, const wave::PackRows &weights, cudaStream_t stream) {
  const cudaError_t err = wave::launch_pack_rows(x, weights, wave::env_knobs().linear_pdl, stream);
  return err == cudaSuccess ? WAVE_OK : cuda_fail(err, "linear: laying out an operand");
}

int operand_map(CUtensorMap *map, const Operand &o, int is_bf16, int box_cols, int box_rows) {
  const uint64_t dims[3] = {static_cast<uint64_t>(o.cols), static_cast<uint64_t>(o.rows), static_cast<uint64_t>(o.matrices)};
  const long long group = o.matrices > 1 ? o.group : o.ld * o.rows; // (read by nobody where there is one matrix)
  const uint64_t strides[2] = {static_cast<uint64_t>(o.ld) * 2, static_cast<uint64_t>(group) * 2};
  const uint32_t box[3] = {static_cast<uint32_t>(box_cols), static_cast<uint32_t>(box_rows), 1};
  return wave::make_tensor_map_16bit(map, is_bf16, o.ptr, 3, dims, strides, box);
}

// The same seen as [matrices][chunks of 64 columns][rows][64], so that a stage of
// an MN-major operand is one copy instead of one for each chunk (a copy keeps the
// loading thread 100 cycles, which with four of them bounded the weight gradient).
// Only where the columns are whole chunks: a chunk is not cut at the row's end.
bool chunked(const Operand &o) { return o.cols % 64 == 0; }
int chunk_map(CUtensorMap *map, const Operand &o, int is_bf16, int box_chunks, int box_rows) {
  const uint64_t dims[4] = {64, static_cast<uint64_t>(o.rows), static_cast<uint64_t>(o.cols / 64),
                            static_cast<uint64_t>(o.matrices)};
  const long long group = o.matrices > 1 ? o.group : o.ld * o.rows;
  const uint64_t strides[3] = {static_cast<uint64_t>(o.ld) * 2, 128, static_cast<uint64_t>(group) * 2};
  const uint32_t box[4] = {64, static_cast<uint32_t>(box_rows), static_cast<uint32_t>(box_chunks), 1};
  return wave::make_tensor_map_16bit(map, is_bf16, o.ptr, 4, dims, strides, box);
}

// ------------------------------------------------------------ tile choice
// What a launch takes is predicted for every tile and split it could have, and
// the cheapest is taken.  Times in us, fitted to 117 problems (1 to 9000 tokens,
// 256 to 12000 features, the three products, up to 64 experts, inputs in turn out
// of L2 and DRAM), each timed in up to 21 variants: the choice is 0.9 % slower than
// the best variant on average and 14 % at worst.
//   base    launch, first loads, teardown
//   stage   64 of the contraction of one whole tile with nothing else in the way
//   epi     a whole tile's epilogue, which hides behind the next tile's stages
struct TileCost {
  int tile; // columns; 512: CTA pair, 256 x 256
  double base, stage, epi;
};
constexpr TileCost kTileCosts[] = {{16, 2.86, 0.24, 0.36}, {32, 3.08, 0.26, 0.65},  {64, 4.59, 0.19, 0.94},
                                   {128, 4.50, 0.33, 1.16}, {256, 5.34, 0.47, 1.45}, {512, 5.54, 0.325, 2.19}};
constexpr int kPairTile = 512;
constexpr double kL2BytesPerUs = 12.4e6; // all SMs together
constexpr double kSplitCost = 2.3;       // the cluster's barriers and the sum over its CTAs, + 0.03 for each
// CTAs that run side by side in clusters of a size (an SM each): clusters do not
// straddle the GPCs, whose SMs are no multiple of every size (measured with
// cudaOccupancyMaxActiveClusters; 148 SMs).
constexpr int kClusterFit[wave::kLinearMaxSplits + 1] = {0, 148, 148, 135, 132, 130, 132, 105, 120};

struct Plan {
  LinearLaunch launch;
  int tile_q, p_blocks, q_blocks, raster_log2, splits, stages;
};

// A product's extents as the tiles see them.
struct Extents {
  Product kind;
  bool grouped;
  long long M;     // tokens
  int matrices, N, K;
  long long p, q, k; // k: of one tile, an expert's share of the rows for its weight gradient
};

struct Candidate {
  int tile, tile_q, splits;
  bool swap;
  long long pb, qb, tiles; // tiles: as many as the launch has to provide for
  double us;
};

// Blocks of `rows` tokens: at most / about.
long long row_blocks_most(const Extents &e, int rows) {
  return e.grouped ? e.M / rows + (e.matrices < e.M ? e.matrices : e.M) : (e.M + rows - 1) / rows;
}
double row_blocks_about(const Extents &e, int rows) {
  if (!e.grouped)
    return static_cast<double>((e.M + rows - 1) / rows);
  const double experts = static_cast<double>(e.matrices < e.M ? e.matrices : e.M);
  const double each = static_cast<double>(e.M) / experts / rows;
  return experts * (each + 0.5 > 1.0 ? each + 0.5 : 1.0);
}

void predict(const Extents &e, const TileCost &t, int sms, Candidate *c) {
  const bool pair = t.tile == kPairTile;
  const int tile_p = pair ? 256 : 128, tile_n = pair ? 256 : t.tile;
  c->pb = (e.p + tile_p - 1) / tile_p;
  c->qb = (e.q + c->tile_q - 1) / c->tile_q;
  double about, width = c->tile_q;
  if (e.kind == Product::kWeightGrad) {
    c->tiles = c->pb * c->qb * e.matrices;
    about = static_cast<double>(c->tiles);
  } else if (c->swap) {
    c->tiles = c->pb * row_blocks_most(e, c->tile_q);
    const double blocks = row_blocks_about(e, c->tile_q);
    about = static_cast<double>(c->pb) * blocks;
    if (pair) {
      width = static_cast<double>(e.M) / blocks + 16.0; // (steps of 32)
      if (width > c->tile_q)
        width = c->tile_q;
    }
  } else {
    c->tiles = c->qb * row_blocks_most(e, tile_p);
    about = static_cast<double>(c->qb) * row_blocks_about(e, tile_p);
  }
  const double fit = (pair ? sms / 2 : sms * (kClusterFit[c->splits] / 148.0));
  const double ctas = about * c->splits, side = ctas < fit ? ctas : fit;
  // (how many tiles the experts' rows make is not known here: two thirds of a last round)
  const double rounds = e.grouped && ctas > fit ? ctas / fit + 0.65 : static_cast<double>(static_cast<long long>((ctas + fit - 1e-6) / fit));
  const long long k_iters = (e.k + 63) / 64;
  const double mine = static_cast<double>((k_iters + c->splits - 1) / c->splits);
  const double bytes = (tile_p + c->tile_q) * 128.0;
  // (a narrower tile saves less time than columns: its other operand is as wide)
  double stage = t.stage * (1.0 - (pair ? 0.38 : 0.54) * (1.0 - static_cast<double>(c->tile_q) / tile_n));
  if (pair && c->swap) // what is loaded and what is multiplied, a quarter each (38 more problems: 2.3 % behind the best, 16 % at worst)
    stage = t.stage * (0.5 + 0.25 * (c->tile_q + width) / tile_n);
  if (stage < 0.17) // the issue of a stage
    stage = 0.17;
  if (stage < bytes * side / kL2BytesPerUs)
    stage = bytes * side / kL2BytesPerUs;
  double epi = t.epi * width / tile_n;
  if (pair && c->swap && epi < 0.8) // two chunks of 32 tokens, however few there are
    epi = 0.8;
  const double each = mine * stage;
  const double base = t.base + epi;
  if (c->splits == 1)
    c->us = base + rounds * (each > epi ? each : epi);
  else
    c->us = base + kSplitCost + 0.03 * c->splits + rounds * each + (rounds - 1.0) * (base - 1.0);
}

Plan make_plan(Product kind, const Shape &s, bool out_f32, int sms) {
  const wave::EnvKnobs env = wave::env_knobs();
  const wave_linear_desc &d = s.d;
  Plan pl{};
  LinearLaunch &l = pl.launch;
  l.a_mn = kind == Product::kWeightGrad;
  l.b_mn = kind != Product::kForward;
  l.out_f32 = out_f32;
  l.pdl = env.linear_pdl;
  Extents e{kind, s.grouped, d.tokens, s.matrices, d.out_features, d.in_features, 0, 0, 0};
  const long long per_expert = (e.M + s.matrices - 1) / s.matrices;
  Candidate best{};
  best.us = -1.0;
  auto consider = [&](const TileCost &t, bool swap, int splits, int tile_q) {
    Candidate c{};
    c.tile = t.tile;
    c.swap = swap;
    c.splits = splits;
    c.tile_q = tile_q;
    predict(e, t, sms, &c);
    // a split launch has a cluster for every tile there could be
    if (splits > 1 && !env.linear_splits && c.tiles * splits > 2ll * kClusterFit[splits])
      return;
    if (best.us < 0.0 || c.us < best.us)
      best = c;
  };
  // Tokens as columns pay while they leave rows of the tensor core's tile empty
  // otherwise; beyond two tiles of them the two ways are the same.
  const bool may_swap = kind == Product::kForward && env.linear_swap != 0 && (env.linear_swap == 1 || per_expert <= 256);
  const bool may_rows = kind != Product::kForward || (env.linear_swap != 1 && (env.linear_swap == 0 || per_expert > 16));
  // CTA pairs take experts' tokens as columns too: a tile has as many as are there.
  const bool pairs_swap = s.grouped && kind != Product::kWeightGrad && !out_f32 && env.linear_swap != 0;
  for (int swap = may_rows ? 0 : 1; swap <= (may_swap || pairs_swap ? 1 : 0); ++swap) {
    const int features = kind == Product::kInputGrad ? e.K : e.N;
    e.p = swap ? features : kind == Product::kWeightGrad ? e.N : e.M;
    e.q = swap ? e.M : kind == Product::kForward ? e.N : e.K;
    e.k = kind == Product::kForward ? e.K : kind == Product::kInputGrad ? e.N : (s.grouped ? per_expert : e.M);
    for (const TileCost &t : kTileCosts) {
      const bool pair = t.tile == kPairTile;
      const int tile_n = pair ? 256 : t.tile;
      if (pair ? swap && !pairs_swap : swap ? !may_swap || t.tile > 128 : t.tile < 64)
        continue;
      if (out_f32 && t.tile > 128)
        continue;
      // the knobs take what they can of their choice
      if (pair ? env.linear_pair == 0 || env.linear_splits > 1 || (pairs_swap && !swap && env.linear_swap == 1)
               : env.linear_pair == 1 && !out_f32 && (!swap || pairs_swap))
        continue;
      const int knob = env.linear_tile;
      if (!pair && knob && (swap ? knob <= 128 : knob >= 64 && !(out_f32 && knob == 256)) && knob != t.tile)
        continue;
      // Columns of no use are left out where the layout allows: tiles of equal
      // width, as few as there can be or up to three more, which can fill a last
      // round of tiles; where not every SM has one, any number (1100 x 2048 x 6848:
      // 256 columns 40.6 us, 160 31.8; 33 more problems with idle SMs: 2.7 % less).
      const int unit = l.b_mn ? (pair ? 128 : 64) : (pair ? 32 : 16);
      const long long least = (e.q + tile_n - 1) / tile_n;
      int before = 0;
      if (pair && swap) { // blocks of up to so many tokens: a stage loads that much of them
        for (int tile_q = 64; tile_q <= 256; tile_q += 32)
          if (!env.linear_columns || tile_q == env.linear_columns)
            consider(t, swap, 1, tile_q);
        continue;
      }
      const int tile_p = pair ? 256 : 128;
      const long long rows = kind == Product::kWeightGrad ? (e.p + tile_p - 1) / tile_p * s.matrices : row_blocks_most(e, tile_p);
      const int most = swap ? 1 : least * rows < (pair ? sms / 2 : sms) ? 24 : l.b_mn ? 1 : 4;
      for (int more = 0; more < most; ++more) {
        const long long n = least + more > 0 ? least + more : 1;
        int tile_q = tile_n;
        if (!(swap && s.grouped)) {
          tile_q = static_cast<int>(round_up((e.q + n - 1) / n, unit));
          tile_q = tile_q > tile_n ? tile_n : tile_q < unit ? unit : tile_q;
        }
        if (env.linear_columns && !(swap && s.grouped))
          tile_q = env.linear_columns / unit * unit < unit ? unit : env.linear_columns > tile_n ? tile_n : env.linear_columns / unit * unit;
        if (more > 0 && tile_q <= tile_n / 2)
          break;
        if (tile_q == before)
          continue;
        before = tile_q;
        if (swap && !knob && t.tile > 16 && tile_q <= t.tile / 2)
          continue; // the next smaller tile does it
        if (env.linear_splits > 0) {
          consider(t, swap, pair ? 1 : env.linear_splits, tile_q);
          continue;
        }
        for (int c : {1, 2, 3, 4, 6, 8})
          if (c == 1 || (!pair && t.tile < 256 && (e.k + 63) / 64 >= 2 * c && (swap || tile_q / 16 >= c)))
            consider(t, swap, c, tile_q);
      }
    }
  }
  if (best.us < 0.0) { // knobs that exclude one another
    e.p = kind == Product::kWeightGrad ? e.N : e.M;
    e.q = kind == Product::kForward ? e.N : e.K;
    consider(kTileCosts[3], false, 1, 128);
  }
  l.swap = best.swap;
  if (l.swap) { // the operands change sides
    l.a_mn = kind == Product::kInputGrad;
    l.b_mn = 0;
  }
  l.pair = best.tile == kPairTile;
  l.tile_n = l.pair ? 256 : best.tile;
  pl.tile_q = best.tile_q;
  pl.splits = best.splits;
  pl.p_blocks = static_cast<int>(best.pb);
  pl.q_blocks = static_cast<int>(best.qb);
  // 2048 rows of tiles share their columns' panel
  pl.raster_log2 = l.pair ? 3 : 4;
  if (l.pair) {
    const long long pairs = sms / 2;
    l.grid = static_cast<int>(2 * (best.tiles < pairs ? (best.tiles > 0 ? best.tiles : 1) : pairs));
    pl.stages = wave::linear_pair_stages(ragged_of(kind, s), s.matrices);
    return pl;
  }
  l.grid = static_cast<int>(pl.splits > 1 ? best.tiles * pl.splits : (best.tiles < sms ? best.tiles : sms));
  if (l.grid < 1)
    l.grid = pl.splits;
  // A CTA with one tile takes no more stages than that has: what it leaves of the
  // SM lets the next kernel of the stream set itself up meanwhile (one token,
  // 2048 x 2048: 12.3 -> 6.5 us).
  pl.stages = wave::linear_max_stages(l.tile_n, l.out_f32, ragged_of(kind, s), s.matrices);
  if (kind != Product::kWeightGrad || !s.grouped) {
    const long long k_ext = kind == Product::kForward ? e.K : kind == Product::kInputGrad ? e.N : e.M;
    const long long need = ((k_ext + 63) / 64 + pl.splits - 1) / pl.splits;
    if ((pl.splits > 1 || best.tiles <= sms) && need < pl.stages)
      pl.stages = need < 3 ? 3 : static_cast<int>(need);
  }
  return pl;
}

// make_plan, with the thread's last choices at hand: a layer is called with the
// same descriptor again and again, and the predictions cost a microsecond.
Plan plan_product(Product kind, const Shape &s, bool out_f32, int sms) {
  struct Entry {
    wave_linear_desc d;
    Product kind;
    int sms;
    unsigned generation;
    bool out_f32, valid;
    Plan plan;
  };
  constexpr int kEntries = 16;
  static thread_local Entry entries[kEntries];
  static thread_local int next = 0;
  const unsigned generation = wave::env_generation();
  for (const Entry &e : entries)
    if (e.valid && e.kind == kind && e.out_f32 == out_f32 && e.sms == sms && e.generation == generation &&
        memcmp(&e.d, &s.d, sizeof s.d) == 0)
      return e.plan;
  Entry &e = entries[next];
  next = (next + 1) % kEntries;
  e.d = s.d;
  e.kind = kind;
  e.out_f32 = out_f32;
  e.sms = sms;
  e.generation = generation;
  e.plan = make_plan(kind, s, out_f32, sms);
  e.valid = true;
  return e.plan;
}

struct Outputs {
  void *D;
  long long ldd, group_d;
  int elem; // bytes
  void *Z;
  const void *R, *bias;
};

int run_product(Product kind, const Shape &s, const Operand &a_tok, const Operand &b_op, const int *offsets, const Outputs &o,
                bool out_f32, int zero_rest, bool beside, int sms, cudaStream_t stream) {
  const wave_linear_desc &d = s.d;
  const Plan pl = plan_product(kind, s, out_f32, sms);
  const LinearLaunch &l = pl.launch;
  LinearParams p{};
  const int is_bf16 = d.io_type == WAVE_BF16;
  // forward: (x, W) or, swapped, (W, x); input gradient: (dz, W); weight gradient: (dz, x)
  const Operand &a = l.swap ? b_op : a_tok;
  const Operand &b = l.swap ? a_tok : b_op;
  const bool weights_a = l.swap, weights_b = kind != Product::kWeightGrad && !l.swap;
  p.group_a = s.grouped && weights_a;
  p.group_b = s.grouped && weights_b;
  if (kind == Product::kForward) {
    p.P = l.swap ? d.out_features : d.tokens;
    p.Q = l.swap ? d.tokens : d.out_features;
    p.K = d.in_features;
  } else if (kind == Product::kInputGrad) {
    p.P = l.swap ? d.in_features : d.tokens;
    p.Q = l.swap ? d.tokens : d.in_features;
    p.K = d.out_features;
  } else {
    p.P = d.out_features;
    p.Q = d.in_features;
    p.K = d.tokens;
  }
  p.ragged = ragged_of(kind, s);
  p.groups = s.matrices;
  p.offsets = s.grouped ? offsets : nullptr;
  p.tile_q = pl.tile_q;
  p.p_blocks = pl.p_blocks;
  p.q_blocks = pl.q_blocks;
  p.raster_log2 = pl.raster_log2;
  // (tokens on the columns: their blocks are the rows of the walk with experts)
  const uint32_t across = static_cast<uint32_t>(l.swap && s.grouped ? pl.p_blocks : pl.q_blocks);
  p.band_tiles = wave::make_fast_div((across > 0 ? across : 1u) << pl.raster_log2);
  p.group_tiles = wave::make_fast_div(static_cast<uint32_t>(pl.p_blocks) * static_cast<uint32_t>(pl.q_blocks > 0 ? pl.q_blocks : 1));
  p.splits = pl.splits;
  p.stages = pl.stages;
  p.is_bf16 = is_bf16;
  p.act = kind == Product::kForward ? d.activation : WAVE_ACT_NONE;
  p.D = o.D;
  p.ldd = o.ldd;
  p.group_d = o.group_d;
  p.Z = o.Z;
  p.ldz = d.ldz;
  p.R = o.R;
  p.ldr = d.ldr;
  p.bias = o.bias;
  p.bias_f32 = d.bias_type == WAVE_F32;
  p.group_bias = s.grouped ? d.out_features : 0;
  p.vec_d = aligned16(o.D) && (o.ldd * o.elem) % 16 == 0 && (o.group_d * o.elem) % 16 == 0;
  p.vec_z = aligned16(o.Z) && d.ldz % 8 == 0;
  p.vec_r = aligned16(o.R) && d.ldr % 8 == 0;
  p.zero_rest = zero_rest;
  p.beside = beside && l.pdl;
  wave::LinearMaps m;
  const int b_cols = l.pair ? pl.tile_q / 2 : pl.tile_q; // of one CTA
  p.chunks_a = l.a_mn && chunked(a);
  p.chunks_b = l.b_mn && chunked(b);
  int rc = p.chunks_a ? chunk_map(&m.a, a, is_bf16, 2, 64) : operand_map(&m.a, a, is_bf16, 64, l.a_mn ? 64 : 128);
  if (rc != WAVE_OK)
    return rc;
  rc = p.chunks_b ? chunk_map(&m.b, b, is_bf16, b_cols / 64, 64) : operand_map(&m.b, b, is_bf16, 64, l.b_mn ? 64 : b_cols);
  if (rc != WAVE_OK)
    return rc;
  // Results leave by TMA where their rows allow it: a store cuts a row at a
  // multiple of 16 bytes, so its length has to be one.  (A split tile's are written
  // in blocks of 16 columns, tokens on columns by other means.)
  m.d = m.z = m.a;
  if (!l.swap && pl.splits == 1) {
    const bool per_group = p.ragged == wave::kRaggedK;
    const uint32_t row_bytes = kind == Product::kForward && !out_f32 ? 64 : 128; // of a chunk of the epilogue
    const uint64_t rows = static_cast<uint64_t>(p.P), cols = static_cast<uint64_t>(p.Q);
    if (p.vec_d && p.Q * o.elem % 16 == 0) {
      const uint64_t dims[3] = {cols, rows, per_group ? static_cast<uint64_t>(s.matrices) : 1};
      const uint64_t row = static_cast<uint64_t>(o.ldd) * o.elem;
      const uint64_t strides[2] = {row, per_group ? static_cast<uint64_t>(o.group_d) * o.elem : row * rows};
      rc = wave::make_tensor_map_store(&m.d, out_f32 ? WAVE_F32 : d.io_type, o.D, dims, strides, row_bytes, 32);
      if (rc != WAVE_OK)
        return rc;
      p.tma_d = 1;
    }
    if (p.Z && p.vec_z && p.Q % 8 == 0) {
      const uint64_t dims[3] = {cols, rows, 1}, row = static_cast<uint64_t>(d.ldz) * 2;
      const uint64_t strides[2] = {row, row * rows};
      if ((rc = wave::make_tensor_map_store(&m.z, d.io_type, o.Z, dims, strides, 64, 32)) != WAVE_OK)
        return rc;
      p.tma_z = 1;
    }
  }
  cudaError_t err = wave::launch_linear(m, p, l, stream);
  return err == cudaSuccess ? WAVE_OK : cuda_fail(err, "linear launch");
}

Operand tokens_by_in(const Shape &s, const void *ptr) {
  return Operand{ptr, s.d.ldx, 0, s.d.tokens, s.d.in_features, 1};
}
Operand weights(const Shape &s, const void *ptr) {
  return Operand{ptr, s.d.ldw, s.d.expert_stride_w, s.d.out_features, s.d.in_features, s.matrices};
}

// Rows of a chunk of the activation gradient: enough chunks for two blocks to an
// SM where the rows allow it, long ones otherwise (fewer partial sums).
int chunk_rows(const Shape &s, int sms) {
  const long long col_blocks = (s.d.out_features + 255) / 256;
  int rows = 128;
  while (rows > 16 && (s.d.tokens / rows) * col_blocks < 2ll * sms)
    rows /= 2;
  while (s.d.tokens / rows + s.matrices > 32768)
    rows *= 2;
  return rows;
}

// Whether a block takes all rows of a group (up to a limit, as the mean is all that
// is known here): one launch instead of two where no group can exceed it, and with
// experts no search for the group of a chunk in each of many blocks.  All rows /
// chunks in us, bf16: what the gradient of gelu or silu and the column sums add to
// dx, 64 x 512 2.4 / 3.7, 128 x 4096 3.0 / 4.4, 250 x 1024 3.6 / 4.0, 500 x 1024 5.4 /
// 4.2; both alone by expert, 24 with 700 rows x 520 in all 3.3 / 5.7, 32 with 3008 x
// 1032 7.9 / 10.1, 64 with 16384 x 1024 21.7 / 24.9, 16 with 4800 x 4096 22.7 / 28.0,
// 16 with 9600 x 4096 38.9 / 43.5 (with dx 105.5 / 105.9: here it ends); one of 16 with
// all of 8192 x 2048, with dx, 58 / 40, and with the mean above it always chunks.
bool short_groups(const Shape &s) {
  const long long rows = (s.d.tokens + s.matrices - 1) / s.matrices;
  return rows <= (s.grouped ? 640 : 256);
}

struct BackwardLayout {
  bool make_dz;   // dz has to be written: an activation, an f32 dy, or rows that TMA cannot load
  long long lddz;
  int chunk;
  bool short_groups;
  bool one_pass; // the activation's gradient and the column sums are one launch
  size_t dz_bytes, partial_bytes, x_bytes, w_bytes;
};
BackwardLayout backward_layout(const Shape &s, int sms) {
  BackwardLayout b{};
  const wave_linear_desc &d = s.d;
  b.make_dz = d.activation != WAVE_ACT_NONE || d.y_type == WAVE_F32 || d.ldy % 8 != 0;
  b.lddz = round_up(d.out_features, 8);
  b.chunk = chunk_rows(s, sms);
  b.dz_bytes = b.make_dz ? static_cast<size_t>(round_up(b.lddz * 2 * d.tokens, 256)) : 0;
  const int groups = s.grouped ? s.matrices : 0;
  b.short_groups = short_groups(s);
  const int more = wave::linear_act_grad_short_more(d.tokens, groups);
  b.one_pass = b.short_groups && more == 0;
  const long long sums = b.one_pass       ? 0
                         : b.short_groups ? groups + more
                                          : wave::linear_act_grad_chunks(d.tokens, groups, b.chunk);
  b.partial_bytes = static_cast<size_t>(round_up(sums * d.out_features * 4ll, 256));
  b.x_bytes = tokens_by_in(s, nullptr).packed_bytes();
  b.w_bytes = weights(s, nullptr).packed_bytes();
  return b;
}

} // namespace

extern "C" {

void wave_cuda_linear_desc_init(wave_linear_desc *d, int tokens, int out_features, int in_features) {
  memset(d, 0, sizeof *d);
  d->tokens = tokens;
  d->out_features = out_features;
  d->in_features = in_features;
  d->io_type = d->y_type = d->bias_type = d->dweight_type = WAVE_BF16;
  d->dbias_type = WAVE_F32;
}

int wave_cuda_linear_validate(const wave_linear_desc *d) { return validate(d); }

int wave_cuda_linear_workspace_bytes(const wave_linear_desc *d, int backward, size_t *bytes) {
  int rc = validate(d);
  if (rc != WAVE_OK)
    return rc;
  if (!bytes)
    return fail(WAVE_E_INVALID, "the result pointer is null");
  const Shape s = resolve(*d);
  if (!backward) {
    *bytes = tokens_by_in(s, nullptr).packed_bytes() + weights(s, nullptr).packed_bytes();
    return WAVE_OK;
  }
  int sms = 0;
  if ((rc = sm_count(&sms)) != WAVE_OK)
    return rc;
  const BackwardLayout b = backward_layout(s, sms);
  *bytes = b.dz_bytes + b.partial_bytes + b.x_bytes + b.w_bytes;
  return WAVE_OK;
}

int wave_cuda_linear_plan_for_sms(const wave_linear_desc *d, int product, int sm_count, wave_linear_plan *plan) {
  const int rc = validate(d);
  if (rc != WAVE_OK)
    return rc;
  if (product < 0 || product > 2 || sm_count < 2 || !plan)
    return fail(WAVE_E_INVALID, "product must be 0 (forward), 1 (input gradient) or 2 (weight gradient), sm_count at least 2 "
                                "and the result pointer non-null; got product=%d, sm_count=%d", product, sm_count);
  const Shape s = resolve(*d);
  const Product kind = product == 0 ? Product::kForward : product == 1 ? Product::kInputGrad : Product::kWeightGrad;
  const bool f32 = product == 0 ? d->y_type == WAVE_F32 : product == 2 && d->dweight_type == WAVE_F32;
  const Plan pl = plan_product(kind, s, f32, sm_count);
  *plan = wave_linear_plan{pl.launch.pair ? 256 : 128, pl.tile_q, pl.launch.swap, pl.splits, pl.launch.grid, pl.stages};
  return WAVE_OK;
}

int wave_cuda_linear_fwd(const wave_linear_desc *d, const void *X, const void *W, const void *bias, const void *residual,
                         const int *offsets, void *Y, void *Z, void *workspace, void *stream) {
  return guarded([&] {
    int rc = validate(d);
    if (rc != WAVE_OK)
      return rc;
    const Shape s = resolve(*d);
    if (s.grouped && !offsets)
      return fail(WAVE_E_INVALID, "grouped layers need the experts' offsets");
    if (s.grouped && residual)
      return fail(WAVE_E_UNSUPPORTED, "a residual goes with one weight matrix, not with experts");
    if (d->tokens == 0)
      return WAVE_OK;
    if (!X || !W || !Y)
      return fail(WAVE_E_INVALID, "X, W and Y must be non-null device pointers");
    if (!aligned16(X) || !aligned16(W))
      return fail(WAVE_E_INVALID, "X and W must be 16-byte aligned");
    if ((rc = check_sum("y", d->y_type, d->in_features)) != WAVE_OK)
      return rc;
    int sms = 0;
    if ((rc = sm_count(&sms)) != WAVE_OK)
      return rc;
    Operand x = tokens_by_in(s, X), w = weights(s, W);
    if (x.packed_bytes() + w.packed_bytes() > 0 && (!workspace || !aligned16(workspace)))
      return fail(WAVE_E_INVALID, "rows of X or W that are no multiple of 16 bytes apart need a 16-byte aligned workspace of %zu bytes",
                  x.packed_bytes() + w.packed_bytes());
    char *ws = static_cast<char *>(workspace);
    cudaStream_t q = static_cast<cudaStream_t>(stream);
    const wave::PackRows px = pack(&x, &ws), pw = pack(&w, &ws, s.grouped ? offsets : nullptr, d->tokens);
    if ((rc = run_packs(px, pw, q)) != WAVE_OK)
      return rc;
    const bool f32 = s.d.y_type == WAVE_F32;
    const Outputs o{Y, s.d.ldy, 0, f32 ? 4 : 2, Z, residual, bias};
    return run_product(Product::kForward, s, x, w, offsets, o, f32, d->zero_rest, false, sms, q);
  });
}

int wave_cuda_linear_bwd(const wave_linear_desc *d, const void *dY, const void *X, const void *W, const void *Z,
                         const int *offsets, void *dX, void *dW, void *dbias, void *workspace, void *stream) {
  return guarded([&] {
    int rc = validate(d);
    if (rc != WAVE_OK)
      return rc;
    const Shape s = resolve(*d);
    if (s.grouped && !offsets)
      return fail(WAVE_E_INVALID, "grouped layers need the experts' offsets");
    if (d->tokens > 0) {
      if (!dY || (dW && !X) || (dX && !W))
        return fail(WAVE_E_INVALID, "dY, the X that dW needs and the W that dX needs must be non-null device pointers");
      if (d->activation != WAVE_ACT_NONE && !Z)
        return fail(WAVE_E_INVALID, "the gradient of an activation needs the pre-activation Z");
      if (!aligned16(dY) || (dW && !aligned16(X)) || (dX && !aligned16(W)))
        return fail(WAVE_E_INVALID, "dY, X and W must be 16-byte aligned");
      if (dX && (rc = check_sum("dX", d->io_type, d->out_features)) != WAVE_OK)
        return rc;
      if (dW && (rc = check_sum("dW", d->dweight_type, d->tokens)) != WAVE_OK)
        return rc;
    }
    int sms = 0;
    if ((rc = sm_count(&sms)) != WAVE_OK)
      return rc;
    const BackwardLayout b = backward_layout(s, sms);
    const size_t need = b.dz_bytes + b.partial_bytes + b.x_bytes + b.w_bytes;
    if (need > 0 && (!workspace || !aligned16(workspace)))
      return fail(WAVE_E_INVALID, "the backward pass needs a 16-byte aligned workspace of %zu bytes", need);
    cudaStream_t q = static_cast<cudaStream_t>(stream);
    char *ws = static_cast<char *>(workspace);
    const int is_bf16 = d->io_type == WAVE_BF16;
    Operand dz{dY, s.d.ldy, 0, s.d.tokens, s.d.out_features, 1};
    const bool dz_wanted = b.make_dz && (dX || dW);
    wave::LinearActGrad g{};
    if (dz_wanted || dbias) {
      g.rows = s.d.tokens;
      g.cols = s.d.out_features;
      g.groups = s.matrices;
      g.offsets = s.grouped ? offsets : nullptr;
      g.act = s.d.activation;
      g.is_bf16 = is_bf16;
      g.dy_f32 = s.d.y_type == WAVE_F32;
      g.dY = dY;
      g.ldy = s.d.ldy;
      g.Z = s.d.activation != WAVE_ACT_NONE ? Z : nullptr;
      g.ldz = s.d.ldz;
      g.dZ = dz_wanted ? ws : nullptr;
      g.lddz = b.lddz;
      g.partial = dbias && !b.one_pass ? reinterpret_cast<float *>(ws + b.dz_bytes) : nullptr;
      g.short_groups = b.short_groups;
      g.short_cols = (d->out_features + 63ll) / 64 * s.matrices >= 2ll * sms ? 64 : 32;
      g.chunk_rows = b.chunk;
      g.dbias = dbias;
      g.dbias_type = s.d.dbias_type == WAVE_F32 ? 0 : is_bf16 ? 2 : 1;
      g.vec_dy = aligned16(dY) && (s.d.ldy * (g.dy_f32 ? 4 : 2)) % 16 == 0;
      g.vec_z = aligned16(g.Z) && s.d.ldz % 8 == 0;
      g.pdl = wave::env_knobs().linear_pdl;
      cudaError_t err = wave::launch_act_grad(g, q);
      if (err == cudaSuccess && dbias && !b.short_groups)
        err = wave::launch_column_sums(g, q);
      if (err != cudaSuccess)
        return cuda_fail(err, "linear: gradient of the activation");
    }
    if (b.make_dz) {
      dz.ptr = ws;
      dz.ld = b.lddz;
    }
    ws += b.dz_bytes + b.partial_bytes;
    Operand w = weights(s, W), x = tokens_by_in(s, X);
    // The products need nothing of the column sums, nor the second product of the first.
    bool beside = dbias && !(dz_wanted && b.short_groups);
    if (s.d.tokens > 0) {
      const wave::PackRows pw = dX ? pack(&w, &ws, s.grouped ? offsets : nullptr, d->tokens) : wave::PackRows{};
      const wave::PackRows px = dW ? pack(&x, &ws) : wave::PackRows{};
      if ((rc = run_packs(px, pw, q)) != WAVE_OK)
        return rc;
      if (pw.groups + px.groups > 0)
        beside = false;
    }
    if (dX && s.d.tokens > 0) {
      const Outputs o{dX, s.d.lddx, 0, 2, nullptr, nullptr, nullptr};
      if ((rc = run_product(Product::kInputGrad, s, dz, w, offsets, o, false, d->zero_rest, beside, sms, q)) != WAVE_OK)
        return rc;
      beside = true;
    }
    if (dW) {
      const bool f32 = s.d.dweight_type == WAVE_F32;
      const Outputs o{dW, s.d.lddw, s.grouped ? s.d.expert_stride_dw : 0, f32 ? 4 : 2, nullptr, nullptr, nullptr};
      if (s.d.tokens == 0) { // no rows: the sums are empty
        cudaError_t err = cudaSuccess;
        const size_t row = static_cast<size_t>(s.d.in_features) * o.elem;
        for (int g = 0; g < s.matrices && err == cudaSuccess; ++g)
          err = cudaMemset2DAsync(static_cast<char *>(dW) + static_cast<size_t>(g) * o.group_d * o.elem,
                                  static_cast<size_t>(s.d.lddw) * o.elem, 0, row, static_cast<size_t>(s.d.out_features), q);
        return err == cudaSuccess ? WAVE_OK : cuda_fail(err, "linear: clearing the weight gradient");
      }
      if ((rc = run_product(Product::kWeightGrad, s, dz, x, offsets, o, f32, 0, beside, sms, q)) != WAVE_OK)
        return rc;
    }
    // Last, as there is seldom anything left of them: in front of the products, which then start later, this launch cost
    // each call 3 to 6 us, here about one.
    if (dbias && b.short_groups && !b.one_pass) {
      cudaError_t err = wave::launch_column_sums(g, q);
      if (err != cudaSuccess)
        return cuda_fail(err, "linear: column sums");
    }
    return WAVE_OK;
  });
}

} // extern "C"
