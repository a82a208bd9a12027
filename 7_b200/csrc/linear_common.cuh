// Device pieces shared by the kernels of the linear layers: the experts' row
// ranges, the walk over the output tiles, the activations and the epilogue.
#pragma once
#include "linear_sm100.h"
#include "sm100_ptx.cuh"

#include <math.h>

namespace wave {
namespace linear_detail {

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

// Executed by all threads of the block; ends with a barrier.
__device__ __forceinline__ void build_group_table(const GroupTable &t, const int *offsets, int groups, int rows,
                                                  int block_rows) {
  for (int i = threadIdx.x; i <= groups; i += blockDim.x)
    t.begin[i] = offsets ? min(max(offsets[i], 0), rows) : (i == 0 ? 0 : rows);
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
      int n = i <= groups && i > 0 ? (v - before + block_rows - 1) / block_rows : 0; // row blocks of group i - 1
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
struct Tile {
  int group;
  int p0, p_end;     // first row on the P side, end of the live rows
  int q0, q_end;     // first column on the Q side, end of the live columns
  int k_begin, k_len; // contraction: first index (rows of the group when ragged) and length
};

// Local tile id -> (row block, column block): `raster` row blocks are walked
// down before the next column block, so that the tiles in flight at one time
// share panels of both operands in L2.
__device__ __forceinline__ void raster_coords(int id, int num_r, int num_c, int raster, int &r, int &c) {
  const int per = raster * num_c;
  const int band = id / per;
  const int first = band * raster;
  const int rows = min(num_r - first, raster);
  const int in = id - band * per;
  r = first + in % rows;
  c = in / rows;
}

template <bool kSwap> struct TileWalk {
  const LinearParams &p;
  const GroupTable t;
  int g;
  int tile_p;
  __device__ TileWalk(const LinearParams &params, const GroupTable &table, int rows_of_tile)
      : p(params), t(table), g(0), tile_p(rows_of_tile) {}
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
      raster_coords(id - t.blocks[g] * other, blocks, other, p.raster, rb, fb);
      w.group = g;
      if (kSwap) {
        w.p0 = fb * tile_p;
        w.p_end = p.P;
        w.q0 = t.begin[g] + rb * p.tile_q;
        w.q_end = t.begin[g + 1];
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
      w.group = id / per;
      if (w.group >= p.groups)
        return false;
      id -= w.group * per;
      w.k_begin = t.begin[w.group];
      w.k_len = t.begin[w.group + 1] - w.k_begin;
    } else if (id >= per) {
      return false;
    }
    raster_coords(id, p.p_blocks, p.q_blocks, p.raster, pb, qb);
    w.p0 = pb * tile_p;
    w.p_end = p.P;
    w.q0 = qb * p.tile_q;
    w.q_end = p.Q;
    return true;
  }
};

// ------------------------------------------------------------- activations
// All in f32 on the unrounded pre-activation.  sigmoid(x) = 1 / (1 + e^-x); the
// exponential is 2^(x log2 e) on the special-function unit (2^-22 relative for
// |x| < 4, 2^-20 at 20: far below a 16-bit rounding and below 2e-6 in f32).
__device__ __forceinline__ float exp_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}

constexpr float kGeluC = 0.7978845608028654f; // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

__device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
  case kActRelu:
    return z < 0.0f ? 0.0f : z; // a NaN stays one
  case kActGelu:
    return 0.5f * z * (1.0f + erff(z * 0.7071067811865476f));
  case kActGeluTanh: // 0.5 z (1 + tanh u) = z sigmoid(2 u)
    return __fdividef(z, 1.0f + exp_fast(-2.0f * kGeluC * (z + kGeluA * z * z * z)));
  case kActSilu:
    return __fdividef(z, 1.0f + exp_fast(-z));
  }
  return z;
}

__device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
  case kActRelu:
    return z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
  case kActGelu:
    return 0.5f * (1.0f + erff(z * 0.7071067811865476f)) + z * 0.3989422804014327f * exp_fast(-0.5f * z * z);
  case kActGeluTanh: {
    const float s = __fdividef(1.0f, 1.0f + exp_fast(-2.0f * kGeluC * (z + kGeluA * z * z * z)));
    return s + z * s * (1.0f - s) * (2.0f * kGeluC) * (1.0f + 3.0f * kGeluA * z * z);
  }
  case kActSilu: {
    const float s = __fdividef(1.0f, 1.0f + exp_fast(-z));
    return s * (1.0f + z * (1.0f - s));
  }
  }
  return 1.0f;
}

// The switch outside the loop over the values.
template <int W> __device__ __forceinline__ void apply_act(float (&v)[W], int act) {
  switch (act) {
  case kActRelu:
#pragma unroll
    for (int i = 0; i < W; ++i)
      v[i] = act_value(v[i], kActRelu);
    break;
  case kActGelu:
#pragma unroll
    for (int i = 0; i < W; ++i)
      v[i] = act_value(v[i], kActGelu);
    break;
  case kActGeluTanh:
#pragma unroll
    for (int i = 0; i < W; ++i)
      v[i] = act_value(v[i], kActGeluTanh);
    break;
  case kActSilu:
#pragma unroll
    for (int i = 0; i < W; ++i)
      v[i] = act_value(v[i], kActSilu);
    break;
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
// places through a slot of shared memory that belongs to the warp: 16 bytes to a
// lane, a row's pieces in neighbouring lanes, whole 32-byte sectors on the way
// out.  The pitch (an odd number of 16-byte units) keeps both directions free of
// bank conflicts.
template <int kElem> __host__ __device__ constexpr int slot_pitch(int cols) { return cols * kElem + 16; }

// Rows [0, rows) x columns [0, cols) of the slot to memory.
template <int kElem, int W>
__device__ __forceinline__ void slot_to_global(const uint8_t *slot, void *base, long long ld, int rows, int cols,
                                               bool vec, int lane) {
  constexpr int kPieces = W * kElem / 16; // of a row
  constexpr int kVals = 16 / kElem;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int idx = i * 32 + lane;
    const int r = idx / kPieces, piece = idx % kPieces;
    const int col = piece * kVals;
    if (r >= rows || col >= cols)
      continue;
    const uint8_t *src = slot + r * slot_pitch<kElem>(W) + piece * 16;
    uint8_t *dst = static_cast<uint8_t *>(base) + (static_cast<long long>(r) * ld + col) * kElem;
    const uint4 v = *reinterpret_cast<const uint4 *>(src);
    if (vec && col + kVals <= cols) {
      *reinterpret_cast<uint4 *>(dst) = v;
    } else {
      const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < kVals; ++e)
        if (col + e < cols) {
          if constexpr (kElem == 4)
            *reinterpret_cast<uint32_t *>(dst + e * 4) = words[e];
          else
            *reinterpret_cast<uint16_t *>(dst + e * 2) = static_cast<uint16_t>(words[e >> 1] >> ((e & 1) * 16));
        }
    }
  }
}

// A 16-bit block of 32 rows x W columns from memory into registers, in the
// order of slot_to_global; what lies outside rows x cols is zero.
template <int W>
__device__ __forceinline__ void global_to_regs(uint4 (&out)[W / 8], const void *base, long long ld, int rows, int cols,
                                               bool vec, int lane) {
  constexpr int kPieces = W / 8;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int idx = i * 32 + lane;
    const int r = idx / kPieces, piece = idx % kPieces;
    const int col = piece * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < rows && col < cols) {
      const uint16_t *src = static_cast<const uint16_t *>(base) + static_cast<long long>(r) * ld + col;
      if (vec && col + 8 <= cols) {
        v = *reinterpret_cast<const uint4 *>(src);
      } else {
        uint32_t words[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (col + e < cols)
            words[e >> 1] |= static_cast<uint32_t>(src[e]) << ((e & 1) * 16);
        v = make_uint4(words[0], words[1], words[2], words[3]);
      }
    }
    out[i] = v;
  }
}
template <int W> __device__ __forceinline__ void regs_to_slot(uint8_t *slot, const uint4 (&v)[W / 8], int lane) {
  constexpr int kPieces = W / 8;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int idx = i * 32 + lane;
    *reinterpret_cast<uint4 *>(slot + (idx / kPieces) * slot_pitch<2>(W) + (idx % kPieces) * 16) = v[i];
  }
}

template <int W> __device__ __forceinline__ void row_to_slot_16bit(uint8_t *slot, const float (&v)[W], int bf16, int lane) {
  uint4 *dst = reinterpret_cast<uint4 *>(slot + lane * slot_pitch<2>(W));
#pragma unroll
  for (int k = 0; k < W / 8; ++k)
    dst[k] = make_uint4(pack_pair(v[8 * k], v[8 * k + 1], bf16), pack_pair(v[8 * k + 2], v[8 * k + 3], bf16),
                        pack_pair(v[8 * k + 4], v[8 * k + 5], bf16), pack_pair(v[8 * k + 6], v[8 * k + 7], bf16));
}

// What a warp's epilogue needs to know of its tile.
struct EpiTile {
  int group;
  int lane0;     // first of the warp's 32 P rows
  int lane_end;  // end of the live P rows
  int q_end;     // end of the live Q columns
};

// Bytes of a warp's slot.
template <bool kF32> __host__ __device__ constexpr int slot_bytes() {
  return 32 * (kF32 ? slot_pitch<4>(32) : slot_pitch<2>(32));
}

// The residual of a chunk, fetched ahead of the accumulator (tokens as rows).
template <int W>
__device__ __forceinline__ void fetch_residual(uint4 (&res)[W / 8], const LinearParams &p, const EpiTile &t, int q0,
                                               int lane) {
  const int rows = min(32, t.lane_end - t.lane0), cols = min(W, t.q_end - q0);
  global_to_regs<W>(res, static_cast<const uint16_t *>(p.R) + static_cast<long long>(t.lane0) * p.ldr + q0, p.ldr, rows,
                    cols, p.vec_r != 0, lane);
}

// Tokens as rows: v holds columns q0 .. q0 + W of the lane's row.
template <bool kF32, int W>
__device__ __forceinline__ void epilogue_rows(const LinearParams &p, const EpiTile &t, int q0, float (&v)[W],
                                              const uint4 (&res)[W / 8], uint8_t *slot, int lane) {
  const int rows = min(32, t.lane_end - t.lane0), cols = min(W, t.q_end - q0);
  if (rows <= 0 || cols <= 0)
    return; // the same for the whole warp
  if (p.bias) {
    // one value to a lane, handed round through the slot
    float b = 0.0f;
    if (lane < cols) {
      const long long at = t.group * p.group_bias + q0 + lane;
      b = p.bias_f32 ? static_cast<const float *>(p.bias)[at]
                     : from_16bit(static_cast<const uint16_t *>(p.bias)[at], p.is_bf16);
    }
    if (lane < W)
      reinterpret_cast<float *>(slot)[lane] = b;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < W / 4; ++k) {
      const float4 f = reinterpret_cast<const float4 *>(slot)[k];
      v[4 * k] += f.x;
      v[4 * k + 1] += f.y;
      v[4 * k + 2] += f.z;
      v[4 * k + 3] += f.w;
    }
    __syncwarp();
  }
  if (p.Z) {
    row_to_slot_16bit<W>(slot, v, p.is_bf16, lane);
    __syncwarp();
    slot_to_global<2, W>(slot, static_cast<uint16_t *>(p.Z) + static_cast<long long>(t.lane0) * p.ldz + q0, p.ldz, rows,
                         cols, p.vec_z != 0, lane);
    __syncwarp();
  }
  apply_act<W>(v, p.act);
  if (p.R) {
    regs_to_slot<W>(slot, res, lane);
    __syncwarp();
    const uint4 *mine = reinterpret_cast<const uint4 *>(slot + lane * slot_pitch<2>(W));
#pragma unroll
    for (int k = 0; k < W / 8; ++k) {
      const uint4 w = mine[k];
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack_pair(words[e], p.is_bf16);
        v[8 * k + 2 * e] += f.x;
        v[8 * k + 2 * e + 1] += f.y;
      }
    }
    __syncwarp(); // f32 rows are longer: the slot may be rewritten once every lane has its residual
  }
  const long long at = t.group * p.group_d + static_cast<long long>(t.lane0) * p.ldd + q0;
  if constexpr (kF32) {
    float4 *dst = reinterpret_cast<float4 *>(slot + lane * slot_pitch<4>(W));
#pragma unroll
    for (int k = 0; k < W / 4; ++k)
      dst[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    __syncwarp();
    slot_to_global<4, W>(slot, static_cast<float *>(p.D) + at, p.ldd, rows, cols, p.vec_d != 0, lane);
  } else {
    row_to_slot_16bit<W>(slot, v, p.is_bf16, lane);
    __syncwarp();
    slot_to_global<2, W>(slot, static_cast<uint16_t *>(p.D) + at, p.ldd, rows, cols, p.vec_d != 0, lane);
  }
  __syncwarp();
}

// Tokens as columns: v[j] is feature `lane0 + lane` of token q0 + j * step; a
// warp's store of one token covers 32 neighbouring features.
template <bool kF32, int W>
__device__ __forceinline__ void epilogue_columns(const LinearParams &p, const EpiTile &t, int q0, int step,
                                                 float (&v)[W], float bias, int lane) {
  const int n = t.lane0 + lane;
  if (n >= t.lane_end)
    return;
#pragma unroll
  for (int j = 0; j < W; ++j)
    v[j] += bias;
  if (p.Z) {
#pragma unroll
    for (int j = 0; j < W; ++j)
      if (q0 + j * step < t.q_end)
        static_cast<uint16_t *>(p.Z)[static_cast<long long>(q0 + j * step) * p.ldz + n] = to_16bit(v[j], p.is_bf16);
  }
  apply_act<W>(v, p.act);
  if (p.R) {
#pragma unroll
    for (int j = 0; j < W; ++j)
      if (q0 + j * step < t.q_end)
        v[j] += from_16bit(static_cast<const uint16_t *>(p.R)[static_cast<long long>(q0 + j * step) * p.ldr + n], p.is_bf16);
  }
#pragma unroll
  for (int j = 0; j < W; ++j)
    if (q0 + j * step < t.q_end) {
      const long long at = static_cast<long long>(q0 + j * step) * p.ldd + n;
      if constexpr (kF32)
        static_cast<float *>(p.D)[at] = v[j];
      else
        static_cast<uint16_t *>(p.D)[at] = to_16bit(v[j], p.is_bf16);
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
