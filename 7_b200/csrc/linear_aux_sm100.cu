// What the products of the linear layers need around them: the gradient of the
// activation with the bias gradient's column sums, and rows laid out for TMA.
#include "linear_common.cuh"

#include <type_traits>

namespace wave {

namespace {

using namespace linear_detail;

// PDL as in the product kernels: set-up may overlap the kernel before this one.
template <typename Kernel, typename... Args>
cudaError_t launch(dim3 grid, int threads, size_t smem, cudaStream_t stream, int pdl, Kernel kernel, const Args &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// ------------------------------------------------------------------- packing
// Eight elements to a thread, neighbouring threads on neighbouring pieces of a
// row; the source may start at any element, so it is read in 4-byte words and put
// together (2 bytes at a time one token over 8192 x 8191 took 79.4 us with its
// product, so 73.5), and written 16 bytes at a time.  Up to two operands of a call
// in one launch: the grid's first x_rows rows are x's, the others one to a matrix
// of the weights.  With experts a block looks first whether its matrix' expert has
// any rows; it takes kPackTurns pieces a thread, so that there are not many blocks
// that only look (64 experts of 1003 x 1021, all with rows / 4 with rows, in us
// with the product: every matrix copied 81 / 61, with a look 1 turn 93 / 46, 4 81 /
// 21, 16 84 / 29).
struct PackTwo {
  PackRows x, weights;
  int x_rows;
};
constexpr int kPackThreads = 256;
constexpr int kPackTurns = 4;
__device__ __forceinline__ uint4 load_piece(const uint16_t *row, int live) {
  uint32_t w[4] = {0, 0, 0, 0};
  if (live < 8) {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < live)
        w[e >> 1] |= static_cast<uint32_t>(row[e]) << ((e & 1) * 16);
  } else {
    // a row that starts within a word is not its matrix' first, so the half in front of it exists; the one behind its
    // last piece may not
    const bool odd = (reinterpret_cast<uintptr_t>(row) & 2) != 0;
    const uint32_t *words = reinterpret_cast<const uint32_t *>(row - odd);
    uint32_t t[5];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      t[e] = words[e];
    t[4] = odd ? row[7] : 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = __funnelshift_r(t[e], t[e + 1], odd ? 16 : 0);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__global__ void __launch_bounds__(kPackThreads) pack_rows_kernel(const __grid_constant__ PackTwo two) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const bool is_x = static_cast<int>(blockIdx.y) < two.x_rows;
  const PackRows &p = is_x ? two.x : two.weights;
  const int g = is_x ? 0 : static_cast<int>(blockIdx.y) - two.x_rows;
  if (p.offsets) {
    // Group g has rows if its end lies behind all that came before it (see build_group_table).
    const int end = min(max(p.offsets[g + 1], 0), p.tokens);
    bool empty = end <= 0;
    for (int i = threadIdx.x; i <= g; i += kPackThreads)
      empty |= min(max(p.offsets[i], 0), p.tokens) >= end;
    if (__syncthreads_or(empty))
      return;
  }
  const int pieces = (p.cols + 7) / 8;
  const long long total = static_cast<long long>(p.rows) * pieces;
  const uint16_t *s = static_cast<const uint16_t *>(p.src) + g * p.group_src;
  uint16_t *d = static_cast<uint16_t *>(p.dst) + g * p.group_dst;
  const long long block = is_x ? blockIdx.y * static_cast<long long>(gridDim.x) + blockIdx.x : blockIdx.x;
  const long long blocks = is_x ? two.x_rows * static_cast<long long>(gridDim.x) : gridDim.x;
  for (long long i = block * kPackThreads + threadIdx.x; i < total; i += blocks * kPackThreads) {
    const long long r = i / pieces;
    const int c = static_cast<int>(i - r * pieces) * 8;
    *reinterpret_cast<uint4 *>(d + r * p.ld_dst + c) = load_piece(s + r * p.ld_src + c, p.cols - c);
  }
}

// -------------------------------------------- activation gradient, column sums
constexpr int kAgThreads = 256;
constexpr int kAgCols = 256;                   // columns of a block, eight to a thread
constexpr int kAgLanes = kAgThreads / (kAgCols / 8); // rows side by side
// Rows in flight for each thread, where the registers of four blocks to an SM are
// to hold them without spilling (8192 x 8192 bf16, gelu_tanh: 2 rows in 80 us, 3 in
// 83, 4 in 110), and elsewhere.
constexpr int kAgUnrollVec = 2, kAgUnroll = 4;
constexpr int kShortRows = 1024; // most rows of a block of the kernel for short groups

struct Eight {
  float v[8];
};

// Eight consecutive values of a row as they lie in memory: 16 bytes, or 32 in f32.
template <bool kF32> struct Raw {
  uint4 w[kF32 ? 2 : 1];
};

// kVec: all eight exist and are aligned; else `live` of them exist and the others are zero.
// kOnce: nobody reads them again, they may leave L2 first.
template <bool kF32, bool kVec, bool kOnce>
__device__ __forceinline__ void load_raw(Raw<kF32> &out, const void *base, long long at, int live) {
  if constexpr (kF32) {
    const uint32_t *src = static_cast<const uint32_t *>(base) + at;
    if constexpr (kVec) {
      out.w[0] = *reinterpret_cast<const uint4 *>(src);
      out.w[1] = *reinterpret_cast<const uint4 *>(src + 4);
    } else {
      uint32_t t[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        t[e] = e < live ? src[e] : 0u;
      out.w[0] = make_uint4(t[0], t[1], t[2], t[3]);
      out.w[1] = make_uint4(t[4], t[5], t[6], t[7]);
    }
  } else {
    const uint16_t *src = static_cast<const uint16_t *>(base) + at;
    if constexpr (kVec) {
      out.w[0] = kOnce ? __ldcs(reinterpret_cast<const uint4 *>(src)) : *reinterpret_cast<const uint4 *>(src);
    } else {
      uint32_t t[4] = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < live)
          t[e >> 1] |= static_cast<uint32_t>(src[e]) << ((e & 1) * 16);
      out.w[0] = make_uint4(t[0], t[1], t[2], t[3]);
    }
  }
}
template <bool kF32> __device__ __forceinline__ Eight values(const Raw<kF32> &r, int bf16) {
  Eight out;
  if constexpr (kF32) {
    const uint32_t w[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w, r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      out.v[e] = __uint_as_float(w[e]);
  } else {
    const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack_pair(w[e], bf16);
      out.v[2 * e] = f.x;
      out.v[2 * e + 1] = f.y;
    }
  }
  return out;
}

// Rows r, r + kLanes, ... below r1 of eight columns: dz written, its column sums added to acc.
template <int kAct, bool kDyF32, bool kVec, bool kOnce, int kLanes, int kUnroll>
__device__ __forceinline__ void act_grad_rows(const LinearActGrad &p, int r, int r1, int col, int live, float (&acc)[8]) {
  for (; r < r1; r += kLanes * kUnroll) {
    Raw<kDyF32> dy_raw[kUnroll];
    Raw<false> z_raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int row = r + u * kLanes;
      if (row < r1) {
        load_raw<kDyF32, kVec, kOnce>(dy_raw[u], p.dY, static_cast<long long>(row) * p.ldy + col, live);
        if constexpr (kAct >= 0)
          load_raw<false, kVec, kOnce>(z_raw[u], p.Z, static_cast<long long>(row) * p.ldz + col, live);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int row = r + u * kLanes;
      if (row >= r1)
        break;
      Eight g = values<kDyF32>(dy_raw[u], p.is_bf16);
      if constexpr (kAct >= 0) {
        const Eight z = values<false>(z_raw[u], p.is_bf16);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float2 d = __fmul2_rn(make_float2(g.v[e], g.v[e + 1]), slope_pair<kAct>(make_float2(z.v[e], z.v[e + 1])));
          g.v[e] = d.x;
          g.v[e + 1] = d.y;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float2 sum = __fadd2_rn(make_float2(acc[e], acc[e + 1]), make_float2(g.v[e], g.v[e + 1]));
        acc[e] = sum.x;
        acc[e + 1] = sum.y;
      }
      if (p.dZ) {
        // rows of dZ are padded to whole 16-byte pieces; columns behind the last are zero (0 * slope(0))
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[e] = pack_pair(g.v[2 * e], g.v[2 * e + 1], p.is_bf16);
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.dZ) + static_cast<long long>(row) * p.lddz + col) =
            make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}
__device__ __forceinline__ void store_dbias(const LinearActGrad &p, int group, int col, float v) {
  const long long at = static_cast<long long>(group) * p.cols + col;
  if (p.dbias_type == 0)
    static_cast<float *>(p.dbias)[at] = v;
  else
    static_cast<uint16_t *>(p.dbias)[at] = to_16bit(v, p.dbias_type == 2);
}

// The group with blocks[g] <= block < blocks[g + 1].
__device__ __forceinline__ int group_of_block(const GroupTable &t, int groups, int block) {
  int lo = 0, hi = groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.blocks[mid] <= block)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// One chunk of rows x 256 columns to a block.  A chunk never crosses a group's
// end, so its column sums go to one group; which rows chunk `blockIdx.y` has
// comes from the offsets, on the device.
// kAct < 0: dz = dy (column sums alone, or a copy in another layout or type).
// The activation is a template argument: chosen for each value at run time it
// costs more than the arithmetic (8192 x 8192 bf16, gelu_tanh: 243 us).
// Bound by memory: what counts is bytes in flight, so rows wait in registers as
// they lie in memory (widened on arrival they took 98 registers and left two
// blocks to an SM: 177 us).  dy and z leave L2 first, so that more of dz is there
// for the products (4096 x 8192, silu, with dx 59.0 -> 55.4 us, 16384 x 2048 56.6 ->
// 53.0); not where dz is dy itself, nor in the kernel for short groups, whose
// neighbours share lines (15 experts, backward 301 -> 310).
template <int kAct, bool kDyF32, bool kVec>
__global__ void __launch_bounds__(kAgThreads, kVec && !kDyF32 ? 4 : 2)
act_grad_kernel(const __grid_constant__ LinearActGrad p) {
  extern __shared__ int ag_smem[];
  __shared__ float sums[kAgLanes][kAgCols];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int r0, r1;
  if (p.offsets) {
    GroupTable t{ag_smem, ag_smem + p.groups + 1};
    build_group_table(t, p.offsets, p.groups, p.rows, p.chunk_rows);
    const int chunk = blockIdx.y;
    if (chunk >= t.blocks[p.groups])
      return;
    const int g = group_of_block(t, p.groups, chunk);
    r0 = t.begin[g] + (chunk - t.blocks[g]) * p.chunk_rows;
    r1 = min(r0 + p.chunk_rows, t.begin[g + 1]);
  } else {
    r0 = static_cast<int>(blockIdx.y) * p.chunk_rows;
    r1 = min(r0 + p.chunk_rows, p.rows);
  }
  const int tc = threadIdx.x % (kAgCols / 8), tr = threadIdx.x / (kAgCols / 8);
  const int col = static_cast<int>(blockIdx.x) * kAgCols + tc * 8;
  const int live = p.cols - col;
  float acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    acc[e] = 0.0f;
  if (live > 0)
    act_grad_rows<kAct, kDyF32, kVec, (kAct >= 0), kAgLanes, (kVec && !kDyF32 ? kAgUnrollVec : kAgUnroll)>(p, r0 + tr, r1, col, live, acc);
  if (!p.partial)
    return;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    sums[tr][tc * 8 + e] = acc[e];
  __syncthreads();
  const int c = static_cast<int>(blockIdx.x) * kAgCols + threadIdx.x;
  if (c < p.cols) {
    float s = 0.0f;
#pragma unroll
    for (int r = 0; r < kAgLanes; ++r)
      s += sums[r][threadIdx.x];
    p.partial[static_cast<long long>(blockIdx.y) * p.cols + c] = s;
  }
}

// The chunks' sums of each group added up: 32 columns x 8 strands of chunks to a
// block, strands joined in order.  Short groups: only a group that took more than
// one block (see act_grad_short_kernel) has anything left to add, and block y of the
// second dimension does it for the group whose first further block is y: there are
// as many of them as further blocks at most, not as many as groups.
__global__ void __launch_bounds__(256) column_sum_kernel(const __grid_constant__ LinearActGrad p) {
  extern __shared__ int ag_smem[];
  __shared__ float sums[8][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int g = blockIdx.y, c0 = 0, c1 = (p.rows + p.chunk_rows - 1) / p.chunk_rows;
  if (p.offsets) {
    GroupTable t{ag_smem, ag_smem + p.groups + 1};
    if (p.short_groups) {
      build_group_table(t, p.offsets, p.groups, p.rows, kShortRows, kShortRows);
      const int more = blockIdx.y;
      if (more >= t.blocks[p.groups])
        return;
      g = group_of_block(t, p.groups, more);
      if (more != t.blocks[g])
        return;
      c0 = p.groups + more;
      c1 = p.groups + t.blocks[g + 1];
    } else {
      build_group_table(t, p.offsets, p.groups, p.rows, p.chunk_rows);
      c0 = t.blocks[g];
      c1 = t.blocks[g + 1];
    }
  }
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const int col = static_cast<int>(blockIdx.x) * 32 + lane;
  float s = 0.0f;
  if (col < p.cols) {
    if (p.short_groups && strand == 0)
      s = p.partial[static_cast<long long>(g) * p.cols + col];
#pragma unroll 4
    for (int c = c0 + strand; c < c1; c += 8)
      s += p.partial[static_cast<long long>(c) * p.cols + col];
  }
  sums[strand][lane] = s;
  __syncthreads();
  if (strand == 0 && col < p.cols) {
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      total += sums[i][lane];
    store_dbias(p, g, col, total);
  }
}

// Short groups: all rows of a group x 32 or 64 columns to a block, dz and the
// finished column sums in one launch, without partial sums in memory.  64 columns
// are whole lines of 128 bytes, which nobody else reads (they leave L2 first); 32
// are for few groups, where there would be too few blocks.  With dx, 32 / 64
// columns in us: 64 groups of 200 rows x 2048 66 / 52, 16 of 300 x 4096 47 / 39, 15
// of 546 x 4096 73 / 67, 32 of 94 x 1032 17.0 / 16.0; one of 250 x 1024 11.1 / 12.6,
// one of 250 x 4096 13.5 / 14.9.
// That the groups are short is known of their mean only.  No block walks more than
// kShortRows rows: blocks of the grid's second dimension behind the groups' own take
// what is left of a longer group, so many rows each, and its column sums are then
// partial, one row of `partial` to a block of that dimension
// (column_sum_kernel).  One expert of 16 with all of 8192 rows x 2048, with dx: 263 us
// without that limit, 57 with it (44 with 512 rows, 87 with 2048); one of 64 with
// 40960 rows 1320 and 207; 16 of 300 x 4096 54.7 and 55.5.
template <int kAct, bool kDyF32, bool kVec, int kCols>
__global__ void __launch_bounds__(kAgThreads) act_grad_short_kernel(const __grid_constant__ LinearActGrad p) {
  extern __shared__ int ag_smem[];
  __shared__ float sums[kAgThreads / 32][kCols];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int y = blockIdx.y;
  int r0 = 0, r1 = p.rows;
  bool finished = true; // the group has no other block
  if (p.offsets) {
    GroupTable t{ag_smem, ag_smem + p.groups + 1};
    build_group_table(t, p.offsets, p.groups, p.rows, kShortRows, kShortRows);
    int g = y, before = 0; // blocks of the group before this one
    if (y >= p.groups) {
      const int more = y - p.groups;
      if (more >= t.blocks[p.groups])
        return;
      g = group_of_block(t, p.groups, more);
      before = 1 + more - t.blocks[g];
    }
    r0 = t.begin[g] + before * kShortRows;
    r1 = min(r0 + kShortRows, t.begin[g + 1]);
    finished = t.blocks[g] == t.blocks[g + 1];
  }
  const int tc = threadIdx.x % (kCols / 8), tr = threadIdx.x / (kCols / 8);
  const int col = static_cast<int>(blockIdx.x) * kCols + tc * 8;
  const int live = p.cols - col;
  float acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    acc[e] = 0.0f;
  if (live > 0)
    act_grad_rows<kAct, kDyF32, kVec, (kAct >= 0 && kCols * 2 >= 128), kAgThreads / (kCols / 8), (kVec && !kDyF32 ? kAgUnrollVec : kAgUnroll)>(p, r0 + tr, r1, col, live, acc);
  if (!p.dbias)
    return;
  // the rows of a warp, then the warps, in order
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int d = kCols / 8; d < 32; d <<= 1)
      acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], d);
  }
  if ((threadIdx.x & 31) < kCols / 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      sums[threadIdx.x / 32][tc * 8 + e] = acc[e];
  }
  __syncthreads();
  const int c = static_cast<int>(blockIdx.x) * kCols + static_cast<int>(threadIdx.x);
  if (threadIdx.x < kCols && c < p.cols) {
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < kAgThreads / 32; ++i)
      total += sums[i][threadIdx.x];
    if (finished)
      store_dbias(p, y, c, total);
    else
      p.partial[static_cast<long long>(y) * p.cols + c] = total;
  }
}

} // namespace

cudaError_t launch_pack_rows(const PackRows &x, const PackRows &weights, int pdl, cudaStream_t stream) {
  auto blocks_of = [](const PackRows &p) { // for a matrix: enough to fill the machine; the rest in the kernel's loop
    const long long each = p.offsets ? kPackThreads * kPackTurns : kPackThreads;
    const long long n = p.groups > 0 ? (static_cast<long long>(p.rows) * ((p.cols + 7) / 8) + each - 1) / each : 0;
    return n < 4096 ? n : 4096ll;
  };
  const long long a = blocks_of(x), b = blocks_of(weights);
  if (a + b == 0)
    return cudaSuccess;
  const long long across = b > 0 ? b : a;
  const int x_rows = static_cast<int>((a + across - 1) / across);
  return launch(dim3(static_cast<unsigned>(across), static_cast<unsigned>(x_rows + weights.groups)), kPackThreads, 0, stream, pdl,
                pack_rows_kernel, PackTwo{x, weights, x_rows});
}

// (a group's further blocks have whole kShortRows of it in front of them)
int linear_act_grad_short_more(int rows, int groups) { return groups == 0 ? 0 : rows / kShortRows; }

int linear_act_grad_chunks(int rows, int groups, int chunk_rows) {
  const int whole = (rows + chunk_rows - 1) / chunk_rows;
  return groups > 0 ? rows / chunk_rows + (groups < rows ? groups : rows) : whole;
}

namespace {
// The instantiation for the call's activation, type of dy and alignment.
template <int kCols, typename Go> void pick_act_grad(const LinearActGrad &p, Go go) {
  auto with = [&](auto f32, auto vec) {
    constexpr bool kF32 = decltype(f32)::value, kVec = decltype(vec)::value;
    switch (p.Z ? p.act : kActNone) {
    case kActRelu: go(act_grad_kernel<kActRelu, kF32, kVec>, act_grad_short_kernel<kActRelu, kF32, kVec, kCols>); break;
    case kActGelu: go(act_grad_kernel<kActGelu, kF32, kVec>, act_grad_short_kernel<kActGelu, kF32, kVec, kCols>); break;
    case kActGeluTanh: go(act_grad_kernel<kActGeluTanh, kF32, kVec>, act_grad_short_kernel<kActGeluTanh, kF32, kVec, kCols>); break;
    case kActSilu: go(act_grad_kernel<kActSilu, kF32, kVec>, act_grad_short_kernel<kActSilu, kF32, kVec, kCols>); break;
    default: go(act_grad_kernel<-1, kF32, kVec>, act_grad_short_kernel<-1, kF32, kVec, kCols>); break;
    }
  };
  const bool vec = p.vec_dy && (!p.Z || p.vec_z) && p.cols % 8 == 0;
  if (p.dy_f32)
    vec ? with(std::true_type{}, std::true_type{}) : with(std::true_type{}, std::false_type{});
  else
    vec ? with(std::false_type{}, std::true_type{}) : with(std::false_type{}, std::false_type{});
}
} // namespace

cudaError_t launch_act_grad(const LinearActGrad &p, cudaStream_t stream) {
  const size_t table = p.offsets ? 2 * sizeof(int) * (static_cast<size_t>(p.groups) + 1) : 0;
  const unsigned groups = static_cast<unsigned>(p.offsets ? p.groups : 1);
  cudaError_t err = cudaSuccess;
  if (p.short_groups) {
    const unsigned more = static_cast<unsigned>(linear_act_grad_short_more(p.rows, p.offsets ? p.groups : 0));
    const dim3 grid(static_cast<unsigned>((p.cols + p.short_cols - 1) / p.short_cols), groups + more);
    auto go = [&](auto, auto kernel) { err = launch(grid, kAgThreads, table, stream, p.pdl, kernel, p); };
    p.short_cols == 64 ? pick_act_grad<64>(p, go) : pick_act_grad<32>(p, go);
    return err;
  }
  const int chunks = linear_act_grad_chunks(p.rows, p.offsets ? p.groups : 0, p.chunk_rows);
  if (chunks > 0) {
    const dim3 grid(static_cast<unsigned>((p.cols + kAgCols - 1) / kAgCols), static_cast<unsigned>(chunks));
    pick_act_grad<32>(p, [&](auto kernel, auto) { err = launch(grid, kAgThreads, table, stream, p.pdl, kernel, p); });
  }
  return err;
}

cudaError_t launch_column_sums(const LinearActGrad &p, cudaStream_t stream) {
  const size_t table = p.offsets ? 2 * sizeof(int) * (static_cast<size_t>(p.groups) + 1) : 0;
  const int y = p.short_groups ? linear_act_grad_short_more(p.rows, p.offsets ? p.groups : 0) : p.offsets ? p.groups : 1;
  if (y == 0)
    return cudaSuccess;
  // (without rows there are no partial sums, but a bias gradient of zero)
  return launch(dim3(static_cast<unsigned>((p.cols + 31) / 32), static_cast<unsigned>(y)), 256, table, stream, p.pdl,
                column_sum_kernel, p);
}

} // namespace wave
