// Device pieces shared by the kernels of the linear layers: the experts' row
// ranges, the walk over the output tiles, the activations and the epilogue.
#pragma once
#include "linear_sm100.h"
#include "slot_turns.h"
#include "sm100_ptx.cuh"

#include <math.h>

namespace wave {
namespace linear_detail {

// The order of launches on the stream.  A kernel waits until the one before it is
// complete, and lets the one after it start as soon as SMs are free.  With
// `beside` it needs nothing that the launch before it writes (that one is of the
// same call and started after everything both of them need was complete): it
// waits only at its end, so that whoever waits for it has waited for both.  So
// the weight gradient's CTAs take the SMs that the input gradient's last round
// leaves idle, and small products run side by side (with it / one after the other,
// in us: 8192 x 8192 x 2048 446 / 466, 515 x 1032 x 776 18.3 / 19.8, 24 experts,
// 700 x 520 x 1288 34.5 / 37.8).
// What a kernel with `beside` reads was written by a grid further back (dz by the
// pass before the launch before it), and griddepcontrol.wait promises visibility
// to the grid that waits, which that one was not in front of.  It rests on this
// instead: the launch before it let it start only behind its own wait (or was
// itself let start so), and the writing grid was complete and its writes performed,
// in L2, before this one's first instruction; and this one reads none of it through L1, which might hold
// something older: operands come by TMA, offsets by loads that go to L2.
__device__ __forceinline__ void start_after_previous(int beside) {
  if (!beside)
    asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void end_after_previous(int beside) {
  if (beside)
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ------------------------------------------------------------- row ranges
// The experts' row ranges in shared memory: begin[g] .. begin[g + 1] are group
// g's rows, blocks[g] the number of row blocks of the groups before it.  What
// the caller's offsets say is taken with a running maximum and cut to [0,
// rows]: offsets that decrease or lie outside give empty groups, never a row
// that two groups share or that does not exist.
struct GroupTable {
  int *begin;  // [groups + 1]
  int *blocks; // [groups + 1]
};

// Executed by all threads of the block; ends with a barrier.  `skip`: so many of a
// group's first rows are in no block.  (The offsets are read past L1, see
// start_after_previous.)
__device__ __forceinline__ void build_group_table(const GroupTable &t, const int *offsets, int groups, int rows,
                                                  int block_rows, int skip = 0) {
  for (int i = threadIdx.x; i <= groups; i += blockDim.x)
    t.begin[i] = offsets ? min(max(__ldcg(offsets + i), 0), rows) : (i == 0 ? 0 : rows);
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int top = 0, count = 0, prev_last = 0;
    for (int base = 0; base <= groups; base += 32) {
      const int i = base + lane;
      int v = i <= groups ? t.begin[i] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d)
          v = max(v, o);
      }
      v = max(v, top);
      int before = __shfl_up_sync(0xffffffffu, v, 1);
      if (lane == 0)
        before = base == 0 ? v : prev_last;
      int n = i <= groups && i > 0 ? (max(v - before - skip, 0) + block_rows - 1) / block_rows : 0; // row blocks of group i - 1
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, n, d);
        if (lane >= d)
          n += o;
      }
      n += count;
      if (i <= groups) {
        t.begin[i] = v;
        t.blocks[i] = n;
      }
      top = prev_last = __shfl_sync(0xffffffffu, v, 31);
      count = __shfl_sync(0xffffffffu, n, 31);
    }
  }
  __syncthreads();
}

// ---------------------------------------------------------------- tile walk
// A value that is the same in the whole warp, said so that the compiler keeps it
// in a uniform register: the instructions that start TMA copies and products
// take their operands from there.
__device__ __forceinline__ int warp_uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

struct Tile {
  int group = 0;
  int p0 = 0, p_end = 0; // first row on the P side, end of the live rows
  int q0 = 0, q_end = 0; // first column on the Q side, end of the live columns
  int n = 0;             // columns of the tile (kEven only)
  int k_begin = 0, k_len = 0; // contraction: first index (rows of the group when ragged) and length
};

// n / d for 0 <= n < 2^31 without a division (the tiles' ids have to be taken
// apart once in each role and tile: with the machine's divisions that took 1000
// cycles, more than the products of a small expert).  m = ceil(2^(31+s) / d),
// s = ceil(log2 d): m d - 2^(31+s) < d <= 2^s, so the error stays below one step.
__device__ __forceinline__ int fast_div(int n, const FastDiv &f) {
  return f.s == 0 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), f.m) >> (f.s - 1));
}
// n / d: below 2^22 a quotient in f32 is off by one at most.
__device__ __forceinline__ int small_div(int n, int d) {
  if (n >= 1 << 22)
    return n / d;
  int q = __float2int_rz(__fdividef(static_cast<float>(n), static_cast<float>(d)));
  const int r = n - q * d;
  q += r >= d ? 1 : r < 0 ? -1 : 0;
  return q;
}

// Local tile id -> (row block, column block): 2^raster_log2 row blocks are
// walked down before the next column block, so that the tiles in flight at one
// time share panels of both operands in L2.
__device__ __forceinline__ void raster_coords(int id, int num_r, const LinearParams &p, int &r, int &c) {
  const int band = fast_div(id, p.band_tiles);
  const int first = band << p.raster_log2;
  const int in = id - band * static_cast<int>(p.band_tiles.d);
  const int rows = min(num_r - first, 1 << p.raster_log2);
  c = rows == 1 << p.raster_log2 ? in >> p.raster_log2 : small_div(in, rows);
  r = first + in - c * rows;
}

// kEven: an expert's tokens are shared out evenly over as few blocks as tile_q
// allows, in steps of 32 columns.
template <bool kSwap, bool kEven = false> struct TileWalk {
  const LinearParams &p;
  const GroupTable t;
  int g;
  int tile_p;
  int even_of = -1, even = 0; // the group whose blocks' width `even` is
  __device__ TileWalk(const LinearParams &params, const GroupTable &table, int rows_of_tile)
      : p(params), t(table), g(0), tile_p(rows_of_tile) {}
  // get() by a whole warp, the answer in uniform registers.
  __device__ bool get_uniform(int id, Tile &w) {
    const bool got = get(id, w);
    w.group = warp_uniform(w.group);
    w.p0 = warp_uniform(w.p0);
    w.q0 = warp_uniform(w.q0);
    w.k_begin = warp_uniform(w.k_begin);
    w.k_len = warp_uniform(w.k_len);
    if (kEven)
      w.n = warp_uniform(w.n);
    return __all_sync(0xffffffffu, got) != 0;
  }
  // Tiles are asked for in increasing order.  False: there is no such tile.
  __device__ bool get(int id, Tile &w) {
    if (p.ragged == kRaggedRows) {
      const int other = kSwap ? p.p_blocks : p.q_blocks;
      while (g < p.groups && id >= t.blocks[g + 1] * other)
        ++g;
      if (g >= p.groups)
        return false;
      int rb, fb;
      const int blocks = t.blocks[g + 1] - t.blocks[g];
      raster_coords(id - t.blocks[g] * other, blocks, p, rb, fb);
      w.group = g;
      if (kSwap) {
        w.p0 = fb * tile_p;
        w.p_end = p.P;
        w.q_end = t.begin[g + 1];
        if (kEven) {
          if (even_of != g) {
            even_of = g;
            even = (small_div(w.q_end - t.begin[g] + blocks - 1, blocks) + 31) & ~31;
          }
          w.n = even;
          w.q0 = t.begin[g] + rb * even;
        } else {
          w.q0 = t.begin[g] + rb * p.tile_q;
        }
      } else {
        w.p0 = t.begin[g] + rb * tile_p;
        w.p_end = t.begin[g + 1];
        w.q0 = fb * p.tile_q;
        w.q_end = p.Q;
      }
      w.k_begin = 0;
      w.k_len = p.K;
      return true;
    }
    const int per = p.p_blocks * p.q_blocks;
    int pb, qb;
    w.group = 0;
    w.k_begin = 0;
    w.k_len = p.K;
    if (p.ragged == kRaggedK) {
      w.group = fast_div(id, p.group_tiles);
      if (w.group >= p.groups)
        return false;
      id -= w.group * per;
      w.k_begin = t.begin[w.group];
      w.k_len = t.begin[w.group + 1] - w.k_begin;
    } else if (id >= per) {
      return false;
    }
    raster_coords(id, p.p_blocks, p, pb, qb);
    w.p0 = pb * tile_p;
    w.p_end = p.P;
    w.q0 = qb * p.tile_q;
    w.q_end = p.Q;
    return true;
  }
};

// ------------------------------------------------------------- the stage ring
// Position in the ring of stages: index, and the parity of its turn.
struct Ring {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void advance(int stages) {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  }
};
// A wait by a whole warp, which gives up together.  `seen`: the barrier was
// already found complete (looked at while the stage before was being issued: the
// look takes as long as the issue of a stage's products).
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag, bool seen) {
  if (seen)
    return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0;
}
// An arrival in another CTA (or this one) that hands over no memory, such as that
// an accumulator has been read out of tensor memory.  With release semantics it
// waits for whatever the thread has written: 1500 to 2500 cycles of every tile.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// warp_wait that also orders what follows behind what the other CTA's threads
// wrote before they arrived.
__device__ __forceinline__ bool warp_wait_cluster(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
  if (!warp_wait(bar, parity, abort_flag, false))
    return false;
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\t"
               "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
               "selp.b32 %0, 1, 0, p;\n\t}"
               : "=r"(ok)
               : "r"(smem_u32(bar)), "r"(parity)
               : "memory"); // (complete already)
  return __all_sync(0xffffffffu, ok != 0) != 0;
}
__device__ __forceinline__ bool warp_peek(uint64_t *bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_test_wait(bar, parity)) != 0;
}

// All 64-column chunks of an operand that is stored with the contraction as its
// slow direction, by one copy: the tensor is seen as [matrices][chunks][rows][64].
__device__ __forceinline__ void tma_load_chunks(void *dst, const CUtensorMap *map, uint64_t *bar, int row, int chunk, int z) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
               " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(row), "r"(chunk), "r"(z)
               : "memory");
}

// ------------------------------------------------------------- activations
// All in f32 on the unrounded pre-activation, two values at a time (one issue
// slot for both).  The epilogue shares its issue slots with nobody, but it has
// to finish a tile while the tensor core works on the next: with erff and one
// value at a time, 8192 x 8192 x 2048 with gelu took 27 us longer than without.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGeluC = 0.7978845608028654f; // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// 1 / (1 + 2^x) of both
__device__ __forceinline__ float2 sigmoid_of_minus(float2 x) {
  const float2 e = __fadd2_rn(make_float2(ex2(x.x), ex2(x.y)), both(1.0f));
  return make_float2(rcp(e.x), rcp(e.y));
}

// The normal distribution's tail behind |z|, and e^(-z^2 / 2).  `a` is |z|, cut at 20
// where both are 0 in f32.  gelu of a negative z is -|z| times the tail, so the tail
// has to be right relative to itself however small it is: e^(-a^2 / 2) is taken out,
// and what is left (the Mills ratio over sqrt(2 pi): 1/2 at 0, falling like 1/a) is
// t P(t), t = 1 / (1 + 0.3 a), with P of degree 7 fitted to the least relative error
// over a = 0 .. 14 (by least squares, reweighted by the error until it was level):
// 1.5e-7, 4.5e-7 with f32 steps.  The exponential adds 2^-22 and 2e-7 * a^2 / 2.
__device__ __forceinline__ void normal_tail(float2 a, float2 &tail, float2 &gauss) {
  const float2 d = __ffma2_rn(a, both(0.3f), both(1.0f));
  const float2 t = make_float2(rcp(d.x), rcp(d.y));
  float2 q = __ffma2_rn(t, both(0.035674758f), both(-0.15720299f));
  q = __ffma2_rn(q, t, both(0.20635334f));
  q = __ffma2_rn(q, t, both(-0.053683452f));
  q = __ffma2_rn(q, t, both(0.12856151f));
  q = __ffma2_rn(q, t, both(0.09991353f));
  q = __ffma2_rn(q, t, both(0.12075395f));
  q = __ffma2_rn(q, t, both(0.1196293f));
  const float2 x = __fmul2_rn(__fmul2_rn(a, a), both(-0.5f * kLog2e));
  gauss = make_float2(ex2(x.x), ex2(x.y));
  tail = __fmul2_rn(__fmul2_rn(q, t), gauss);
}

template <int kAct> __device__ __forceinline__ float2 act_pair(float2 z) {
  if constexpr (kAct == kActRelu) {
    return make_float2(z.x < 0.0f ? 0.0f : z.x, z.y < 0.0f ? 0.0f : z.y); // a NaN stays one
  } else if constexpr (kAct == kActGelu) {
    // z Phi(z) = max(z, 0) - |z| tail
    const float2 a = make_float2(fminf(fabsf(z.x), 20.0f), fminf(fabsf(z.y), 20.0f));
    float2 tail, gauss;
    normal_tail(a, tail, gauss);
    const float2 top = make_float2(z.x < 0.0f ? 0.0f : z.x, z.y < 0.0f ? 0.0f : z.y);
    return __ffma2_rn(make_float2(-a.x, -a.y), tail, top);
  } else if constexpr (kAct == kActGeluTanh) {
    // 0.5 z (1 + tanh u) = z sigmoid(2 u)
    const float2 k = __ffma2_rn(__fmul2_rn(z, z), both(-2.0f * kLog2e * kGeluC * kGeluA), both(-2.0f * kLog2e * kGeluC));
    return __fmul2_rn(z, sigmoid_of_minus(__fmul2_rn(z, k)));
  } else if constexpr (kAct == kActSilu) {
    return __fmul2_rn(z, sigmoid_of_minus(__fmul2_rn(z, both(-kLog2e))));
  } else {
    return z;
  }
}

template <int kAct> __device__ __forceinline__ float2 slope_pair(float2 z) {
  if constexpr (kAct == kActRelu) {
    return make_float2(z.x > 0.0f ? 1.0f : (z.x <= 0.0f ? 0.0f : z.x), z.y > 0.0f ? 1.0f : (z.y <= 0.0f ? 0.0f : z.y));
  } else if constexpr (kAct == kActGelu) {
    // Phi(z) + z phi(z)
    const float2 a = make_float2(fminf(fabsf(z.x), 20.0f), fminf(fabsf(z.y), 20.0f));
    float2 tail, gauss;
    normal_tail(a, tail, gauss);
    const float2 phi = make_float2(z.x < 0.0f ? tail.x : 1.0f - tail.x, z.y < 0.0f ? tail.y : 1.0f - tail.y);
    const float2 zc = make_float2(z.x < 0.0f ? -a.x : (z.x >= 0.0f ? a.x : z.x), z.y < 0.0f ? -a.y : (z.y >= 0.0f ? a.y : z.y));
    return __ffma2_rn(__fmul2_rn(zc, both(0.3989422804014327f)), gauss, phi);
  } else if constexpr (kAct == kActGeluTanh || kAct == kActSilu) {
    // z s with s = sigmoid(r z), r = 1 or 2c (1 + a z^2): s + z s (1 - s) (r z)' = s (1 + (1 - s) z (r z)').
    // Beyond +-128 (+-16) that is 1 or 0 in f32; cut there, lest (1 - s) z becomes 0 * infinity.
    constexpr float kCutAt = kAct == kActSilu ? 128.0f : 16.0f;
    const float2 c = make_float2(fminf(fmaxf(z.x, -kCutAt), kCutAt), fminf(fmaxf(z.y, -kCutAt), kCutAt));
    float2 s, w;
    if constexpr (kAct == kActSilu) {
      s = sigmoid_of_minus(__fmul2_rn(c, both(-kLog2e)));
      w = c;
    } else {
      const float2 z2 = __fmul2_rn(c, c);
      s = sigmoid_of_minus(__fmul2_rn(c, __ffma2_rn(z2, both(-2.0f * kLog2e * kGeluC * kGeluA), both(-2.0f * kLog2e * kGeluC))));
      w = __fmul2_rn(c, __ffma2_rn(z2, both(6.0f * kGeluC * kGeluA), both(2.0f * kGeluC)));
    }
    const float2 rest = __ffma2_rn(s, both(-1.0f), both(1.0f));
    const float2 y = __fmul2_rn(s, __ffma2_rn(rest, w, both(1.0f)));
    return make_float2(z.x == z.x ? y.x : z.x, z.y == z.y ? y.y : z.y); // a NaN stays one
  } else {
    return both(1.0f);
  }
}

// The switch outside the loop over the values.
template <int kAct, int W> __device__ __forceinline__ void apply_one(float (&v)[W]) {
#pragma unroll
  for (int i = 0; i < W; i += 2) {
    const float2 y = act_pair<kAct>(make_float2(v[i], v[i + 1]));
    v[i] = y.x;
    v[i + 1] = y.y;
  }
}
template <int W> __device__ __forceinline__ void apply_act(float (&v)[W], int act) {
  switch (act) {
  case kActRelu: apply_one<kActRelu, W>(v); break;
  case kActGelu: apply_one<kActGelu, W>(v); break;
  case kActGeluTanh: apply_one<kActGeluTanh, W>(v); break;
  case kActSilu: apply_one<kActSilu, W>(v); break;
  }
}

// ------------------------------------------------------------- 16-bit values
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, int bf16) {
  if (bf16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&v);
  }
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&v);
}
__device__ __forceinline__ float2 unpack_pair(uint32_t w, int bf16) {
  if (bf16)
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<__half2 *>(&w));
}
__device__ __forceinline__ uint16_t to_16bit(float v, int bf16) {
  if (bf16) {
    __nv_bfloat16 b = __float2bfloat16_rn(v);
    return *reinterpret_cast<uint16_t *>(&b);
  }
  __half h = __float2half_rn(v);
  return *reinterpret_cast<uint16_t *>(&h);
}
__device__ __forceinline__ float from_16bit(uint16_t w, int bf16) {
  if (bf16)
    return __uint_as_float(static_cast<uint32_t>(w) << 16);
  return __half2float(*reinterpret_cast<__half *>(&w));
}

// -------------------------------------------------------------- the epilogue
// A warp holds W consecutive columns of 32 rows, one row to a lane, as they come
// out of tensor memory.  Rows of memory are longer than that, so values change
// places through a slot of shared memory that belongs to the warp: 16-byte
// pieces, a row's in neighbouring lanes, whole 32-byte sectors on the way out.
// Piece `c` of row `r` lies at a place that is turned by the row's number, so
// that eight lanes that go down a column of pieces and eight that go along the
// rows both meet all 32 banks.
template <int kElem, int W> struct Slot {
  static constexpr int kPieces = W * kElem / 16; // of a row: 2, 4 or 8
  static constexpr int kVals = 16 / kElem;
  static constexpr int kRowsPerLine = 8 / kPieces; // rows in 128 bytes
  static constexpr int kBytes = 32 * kPieces * 16;
  static_assert(kPieces == 2 || kPieces == 4 || kPieces == 8, "rows of 32, 64 or 128 bytes");
  static __device__ __forceinline__ int at(int r, int c) {
    return (r * kPieces + (c ^ ((r / kRowsPerLine) & (kPieces - 1)))) * 16;
  }
};

// Rows [0, rows) x columns [0, cols) of the slot to memory; `base` is the
// element of row 0, column 0.
template <int kElem, int W>
__device__ __forceinline__ void slot_to_global(const uint8_t *slot, void *base, long long ld, int rows, int cols,
                                               bool vec, int lane) {
  using S = Slot<kElem, W>;
  constexpr int kRowStep = 32 / S::kPieces;
  const int r0 = lane / S::kPieces, piece = lane % S::kPieces;
  uint8_t *dst = static_cast<uint8_t *>(base) + static_cast<long long>(r0) * ld * kElem + piece * 16;
  const long long step = ld * (kRowStep * kElem);
  if (vec && rows == 32 && cols == W) { // the same for the whole warp
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i, dst += step)
      *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(slot + S::at(r0 + i * kRowStep, piece));
    return;
  }
  if (vec) {
    const int live = cols - piece * S::kVals; // columns of the piece that exist
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i, dst += step) {
      if (r0 + i * kRowStep >= rows || live <= 0)
        continue;
      const uint4 v = *reinterpret_cast<const uint4 *>(slot + S::at(r0 + i * kRowStep, piece));
      if (live >= S::kVals) {
        *reinterpret_cast<uint4 *>(dst) = v;
      } else {
        const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < S::kVals; ++e)
          if (e < live) {
            if constexpr (kElem == 4)
              *reinterpret_cast<uint32_t *>(dst + e * 4) = words[e];
            else
              *reinterpret_cast<uint16_t *>(dst + e * 2) = static_cast<uint16_t>(words[e >> 1] >> ((e & 1) * 16));
          }
      }
    }
    return;
  }
  // Rows that start anywhere: a row at a time, a value to a lane, so that a store
  // still covers one piece of memory (a lane's 16 bytes in 2-byte stores scatter
  // over eight rows each: 4000 x 2500 x 1000 took 72 us).
#pragma unroll 8
  for (int r = 0; r < rows; ++r) {
    uint8_t *row = static_cast<uint8_t *>(base) + static_cast<long long>(r) * ld * kElem;
#pragma unroll
    for (int c = lane; c < W; c += 32)
      if (c < cols) {
        const uint8_t *src = slot + S::at(r, c / S::kVals) + c % S::kVals * kElem;
        if constexpr (kElem == 4)
          *reinterpret_cast<uint32_t *>(row + c * 4) = *reinterpret_cast<const uint32_t *>(src);
        else
          *reinterpret_cast<uint16_t *>(row + c * 2) = *reinterpret_cast<const uint16_t *>(src);
      }
  }
}

// A 16-bit block of 32 rows x W columns whose rows are 16-byte aligned from memory
// into registers, in the order of slot_to_global; what lies outside rows x cols is
// zero.
template <int W>
__device__ __forceinline__ void global_to_regs(uint4 (&out)[W / 8], const void *base, long long ld, int rows, int cols,
                                               int lane) {
  using S = Slot<2, W>;
  constexpr int kRowStep = 32 / S::kPieces;
  const int r0 = lane / S::kPieces, piece = lane % S::kPieces;
  const uint16_t *src = static_cast<const uint16_t *>(base) + static_cast<long long>(r0) * ld + piece * 8;
  const long long step = ld * kRowStep;
  if (rows == 32 && cols == W) {
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i, src += step)
      out[i] = *reinterpret_cast<const uint4 *>(src);
    return;
  }
  const int live = cols - piece * 8;
#pragma unroll
  for (int i = 0; i < S::kPieces; ++i, src += step) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r0 + i * kRowStep < rows && live > 0) {
      if (live >= 8) {
        v = *reinterpret_cast<const uint4 *>(src);
      } else {
        uint32_t words[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < live)
            words[e >> 1] |= static_cast<uint32_t>(src[e]) << ((e & 1) * 16);
        v = make_uint4(words[0], words[1], words[2], words[3]);
      }
    }
    out[i] = v;
  }
}
// The same into the slot: from those registers, or straight from memory, a row at
// a time, where the rows start anywhere.
template <int W>
__device__ __forceinline__ void residual_to_slot(uint8_t *slot, const uint4 (&regs)[W / 8], const void *base, long long ld,
                                                 int rows, int cols, bool vec, int lane) {
  using S = Slot<2, W>;
  if (vec) {
    constexpr int kRowStep = 32 / S::kPieces;
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i)
      *reinterpret_cast<uint4 *>(slot + S::at(lane / S::kPieces + i * kRowStep, lane % S::kPieces)) = regs[i];
    return;
  }
#pragma unroll 8
  for (int r = 0; r < rows; ++r) {
    const uint16_t *row = static_cast<const uint16_t *>(base) + static_cast<long long>(r) * ld;
#pragma unroll
    for (int c = lane; c < W; c += 32)
      if (c < cols)
        *reinterpret_cast<uint16_t *>(slot + S::at(r, c / 8) + c % 8 * 2) = row[c];
  }
}

template <int W, bool kBf16> __device__ __forceinline__ void row_to_slot_type(uint8_t *slot, const float (&v)[W], int lane) {
#pragma unroll
  for (int k = 0; k < W / 8; ++k)
    *reinterpret_cast<uint4 *>(slot + Slot<2, W>::at(lane, k)) =
        make_uint4(pack_pair(v[8 * k], v[8 * k + 1], kBf16), pack_pair(v[8 * k + 2], v[8 * k + 3], kBf16),
                   pack_pair(v[8 * k + 4], v[8 * k + 5], kBf16), pack_pair(v[8 * k + 6], v[8 * k + 7], kBf16));
}
template <int W> __device__ __forceinline__ void row_to_slot_16bit(uint8_t *slot, const float (&v)[W], int bf16, int lane) {
  if (bf16) // outside the loop
    row_to_slot_type<W, true>(slot, v, lane);
  else
    row_to_slot_type<W, false>(slot, v, lane);
}
// The residual of the lane's row, as it lies in the slot, added to v.
template <int W, bool kBf16> __device__ __forceinline__ void add_row_from_slot(float (&v)[W], const uint8_t *slot, int lane) {
#pragma unroll
  for (int k = 0; k < W / 8; ++k) {
    const uint4 w = *reinterpret_cast<const uint4 *>(slot + Slot<2, W>::at(lane, k));
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = 8 * k + 2 * e;
      const float2 sum = __fadd2_rn(make_float2(v[j], v[j + 1]), unpack_pair(words[e], kBf16));
      v[j] = sum.x;
      v[j + 1] = sum.y;
    }
  }
}

// What a warp's epilogue needs to know of its tile.
struct EpiTile {
  int group;
  int lane0;     // first of the warp's 32 P rows
  int lane_end;  // end of the live P rows
  int q_end;     // end of the live Q columns
};

// Bytes of a warp's slot: 32 rows of 128.
constexpr int kSlotBytes = 4096;

// What a chunk's epilogue reads from memory, fetched while the chunk before it
// is worked on (tokens as rows): the residual in the order of slot_to_global,
// and the bias, one value to a lane.
template <int W> struct Ahead {
  uint4 res[W / 8];
  float bias[(W + 31) / 32];
};
template <int W>
__device__ __forceinline__ void fetch_ahead(Ahead<W> &f, const LinearParams &p, const EpiTile &t, int q0, int lane) {
  const int rows = min(32, t.lane_end - t.lane0), cols = min(W, t.q_end - q0);
  if (p.R && p.vec_r)
    global_to_regs<W>(f.res, static_cast<const uint16_t *>(p.R) + static_cast<long long>(t.lane0) * p.ldr + q0, p.ldr, rows,
                      cols, lane);
#pragma unroll
  for (int i = 0; i < (W + 31) / 32; ++i) {
    f.bias[i] = 0.0f;
    if (p.bias && lane + 32 * i < cols) {
      const long long at = t.group * p.group_bias + q0 + lane + 32 * i;
      f.bias[i] = p.bias_f32 ? static_cast<const float *>(p.bias)[at]
                             : from_16bit(static_cast<const uint16_t *>(p.bias)[at], p.is_bf16);
    }
  }
}

// What an epilogue warp has of its own: its slot and the
// tensor maps of D and z (their boxes are what it takes: 32 rows).
//
// Blocks leave the slot by one TMA store where they can: through the load-store
// unit a block is read from shared memory and written to L1 a second time, which
// bounds tiles of short sums (the f32 weight gradients of 24 experts with 29 rows
// each: 3100 of a tile's 5500 cycles).  The store cuts what lies behind the
// tensor's last row or column; only a block that ends at an expert's last row has
// to be written row by row.
// Blocks of 64 bytes a row (the forward pass in 16 bits: 32 columns, whose
// arithmetic needs the registers) take the slot's halves in turn, so that one is
// filled while a store reads the other; rows of 128 bytes take it whole.
struct EpiWarp {
  uint8_t *slot;
  const CUtensorMap *map_d, *map_z;
  int lane;
  int other_half = kSlotBytes / 2; // from the half in use to the other
};
// The bulk groups of a warp's stores: lane 0 issues them all.
struct LaneZeroBulk {
  int lane;
  template <int N> __device__ __forceinline__ void wait_read() const {
    if (lane == 0)
      tma_store_wait_read<N>();
  }
  __device__ __forceinline__ void commit() const {
    if (lane == 0)
      tma_store_commit();
  }
};
// Takes the slot, or its other half: the stores that read it have done so.  Each
// slot_next is followed by one slot_out.
template <bool kHalves> __device__ __forceinline__ void slot_next(EpiWarp &e) {
  slot_take<kHalves>(e.slot, e.other_half, LaneZeroBulk{e.lane});
  __syncwarp();
}
template <int kElem, int W>
__device__ __forceinline__ void slot_out(const EpiWarp &e, const CUtensorMap *map, bool tma, void *base, long long ld, int rows,
                                         int cols, bool vec, int q0, int p0, int group) {
  if (W * kElem >= 64 && tma) {
    fence_proxy_async_smem();
    __syncwarp();
    if (e.lane == 0)
      tma_store_3d(map, e.slot, q0, p0, group);
  } else {
    __syncwarp();
    slot_to_global<kElem, W>(e.slot, base, ld, rows, cols, vec, e.lane);
    __syncwarp();
  }
  slot_leave(LaneZeroBulk{e.lane});
}

// Tokens as rows: v holds columns q0 .. q0 + W of the lane's row.  kFull: the
// forward pass; the products of the backward pass only store.
template <bool kF32, int W, bool kFull>
__device__ __forceinline__ void epilogue_rows(const LinearParams &p, const EpiTile &t, int q0, float (&v)[W],
                                              const Ahead<W> &f, EpiWarp &e) {
  constexpr bool kHalves = !kF32 && W * 2 == 64;
  const int lane = e.lane;
  const int rows = min(32, t.lane_end - t.lane0), cols = min(W, t.q_end - q0);
  if (rows <= 0 || cols <= 0)
    return; // the same for the whole warp
  // No row behind these is another expert's, no column another tile's.
  const bool whole = (rows == 32 || p.ragged != kRaggedRows) && (q0 + W <= t.q_end || t.q_end == p.Q);
  if (kFull && p.bias) { // a lane's value handed round (through shared memory it would take a place in the ring of stages)
#pragma unroll
    for (int j = 0; j < W; j += 2) {
      const float2 sum = __fadd2_rn(make_float2(v[j], v[j + 1]), make_float2(__shfl_sync(0xffffffffu, f.bias[j / 32], j % 32),
                                                                             __shfl_sync(0xffffffffu, f.bias[j / 32], j % 32 + 1)));
      v[j] = sum.x;
      v[j + 1] = sum.y;
    }
  }
  if (kFull && p.Z) {
    slot_next<kHalves>(e);
    row_to_slot_16bit<W>(e.slot, v, p.is_bf16, lane);
    slot_out<2, W>(e, e.map_z, p.tma_z && whole, static_cast<uint16_t *>(p.Z) + static_cast<long long>(t.lane0) * p.ldz + q0,
                   p.ldz, rows, cols, p.vec_z != 0, q0, t.lane0, 0);
  }
  if constexpr (kFull)
    apply_act<W>(v, p.act);
  slot_next<kHalves>(e);
  uint8_t *slot = e.slot;
  if (kFull && p.R) {
    residual_to_slot<W>(slot, f.res, static_cast<const uint16_t *>(p.R) + static_cast<long long>(t.lane0) * p.ldr + q0, p.ldr,
                        rows, cols, p.vec_r != 0, lane);
    __syncwarp();
    if (p.is_bf16)
      add_row_from_slot<W, true>(v, slot, lane);
    else
      add_row_from_slot<W, false>(v, slot, lane);
    __syncwarp(); // f32 rows are longer: the slot may be rewritten once every lane has its residual
  }
  const long long at = t.group * p.group_d + static_cast<long long>(t.lane0) * p.ldd + q0;
  if constexpr (kF32) {
#pragma unroll
    for (int k = 0; k < W / 4; ++k)
      *reinterpret_cast<float4 *>(slot + Slot<4, W>::at(lane, k)) =
          make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    slot_out<4, W>(e, e.map_d, p.tma_d && whole, static_cast<float *>(p.D) + at, p.ldd, rows, cols, p.vec_d != 0, q0, t.lane0,
                   p.ragged == kRaggedK ? t.group : 0);
  } else {
    row_to_slot_16bit<W>(slot, v, p.is_bf16, lane);
    slot_out<2, W>(e, e.map_d, p.tma_d && whole, static_cast<uint16_t *>(p.D) + at, p.ldd, rows, cols, p.vec_d != 0, q0, t.lane0,
                   p.ragged == kRaggedK ? t.group : 0);
  }
}

// Tokens as columns: v[j] is feature `lane0 + lane` of token q0 + j.  A few tokens
// are stored as they are, 32 neighbouring features to a store; more change places
// in the warp's slot (a token to a row) and leave as 16-byte pieces.
template <bool kF32, int W>
__device__ __forceinline__ void epilogue_columns(const LinearParams &p, const EpiTile &t, int q0, float (&v)[W],
                                                 float bias, uint8_t *slot, int lane) {
  const int n = t.lane0 + lane;
  const int tokens = min(W, t.q_end - q0), features = min(32, t.lane_end - t.lane0);
  if (tokens <= 0 || features <= 0)
    return; // the same for the whole warp
  const bool staged = W > 8 && tokens > 8;
#pragma unroll
  for (int j = 0; j < W; ++j)
    v[j] += bias;
  if (staged) {
    // the lane's place in row j of the slot
    auto place = [&](int elem, int j) {
      return elem == 4 ? Slot<4, 32>::at(j, lane >> 2) + (lane & 3) * 4 : Slot<2, 32>::at(j, lane >> 3) + (lane & 7) * 2;
    };
    if (p.Z) {
#pragma unroll
      for (int j = 0; j < W; ++j)
        *reinterpret_cast<uint16_t *>(slot + place(2, j)) = to_16bit(v[j], p.is_bf16);
      __syncwarp();
      slot_to_global<2, 32>(slot, static_cast<uint16_t *>(p.Z) + static_cast<long long>(q0) * p.ldz + t.lane0, p.ldz, tokens,
                            features, p.vec_z != 0, lane);
      __syncwarp();
    }
    apply_act<W>(v, p.act);
    if (p.R) {
      const uint16_t *base = static_cast<const uint16_t *>(p.R) + static_cast<long long>(q0) * p.ldr + t.lane0;
      uint4 res[4];
      if (p.vec_r)
        global_to_regs<32>(res, base, p.ldr, tokens, features, lane);
      residual_to_slot<32>(slot, res, base, p.ldr, tokens, features, p.vec_r != 0, lane);
      __syncwarp();
#pragma unroll
      for (int j = 0; j < W; ++j)
        v[j] += from_16bit(*reinterpret_cast<const uint16_t *>(slot + place(2, j)), p.is_bf16);
      __syncwarp();
    }
#pragma unroll
    for (int j = 0; j < W; ++j) {
      if constexpr (kF32)
        *reinterpret_cast<float *>(slot + place(4, j)) = v[j];
      else
        *reinterpret_cast<uint16_t *>(slot + place(2, j)) = to_16bit(v[j], p.is_bf16);
    }
    __syncwarp();
    uint8_t *base = static_cast<uint8_t *>(p.D) + (static_cast<long long>(q0) * p.ldd + t.lane0) * (kF32 ? 4 : 2);
    slot_to_global<kF32 ? 4 : 2, 32>(slot, base, p.ldd, tokens, features, p.vec_d != 0, lane);
    __syncwarp();
    return;
  }
  if (lane >= features)
    return;
  if (p.Z) {
    uint16_t *z = static_cast<uint16_t *>(p.Z) + static_cast<long long>(q0) * p.ldz + n;
#pragma unroll
    for (int j = 0; j < W && j < 8; ++j, z += p.ldz)
      if (j < tokens)
        *z = to_16bit(v[j], p.is_bf16);
  }
  apply_act<W>(v, p.act);
  if (p.R) {
    const uint16_t *r = static_cast<const uint16_t *>(p.R) + static_cast<long long>(q0) * p.ldr + n;
#pragma unroll
    for (int j = 0; j < W && j < 8; ++j, r += p.ldr)
      if (j < tokens)
        v[j] += from_16bit(*r, p.is_bf16);
  }
  uint8_t *d = static_cast<uint8_t *>(p.D) + (static_cast<long long>(q0) * p.ldd + n) * (kF32 ? 4 : 2);
#pragma unroll
  for (int j = 0; j < W && j < 8; ++j, d += p.ldd * (kF32 ? 4 : 2))
    if (j < tokens) {
      if constexpr (kF32)
        *reinterpret_cast<float *>(d) = v[j];
      else
        *reinterpret_cast<uint16_t *>(d) = to_16bit(v[j], p.is_bf16);
    }
}
__device__ __forceinline__ float column_bias(const LinearParams &p, const EpiTile &t, int lane) {
  const int n = t.lane0 + lane;
  if (!p.bias || n >= t.lane_end)
    return 0.0f;
  const long long at = t.group * p.group_bias + n;
  return p.bias_f32 ? static_cast<const float *>(p.bias)[at]
                    : from_16bit(static_cast<const uint16_t *>(p.bias)[at], p.is_bf16);
}

// Rows that belong to no group, set to zero: warp `w` of `warps` over the whole grid.
__device__ __forceinline__ void zero_rows(void *base, int elem, long long ld, int first, int last, int cols, int w,
                                          int warps, int lane) {
  for (int r = first + w; r < last; r += warps) {
    uint8_t *row = static_cast<uint8_t *>(base) + static_cast<long long>(r) * ld * elem;
    for (int c = lane; c < cols; c += 32) {
      if (elem == 4)
        reinterpret_cast<float *>(row)[c] = 0.0f;
      else
        reinterpret_cast<uint16_t *>(row)[c] = 0;
    }
  }
}

} // namespace linear_detail
} // namespace wave
