// Products of the linear layers on one CTA: D = act(A * B^T + bias) + residual,
// dense or grouped by expert, and the two products of the backward pass.
//
// One 128 x TN tile at a time: TMA fills a ring of 64-deep stages (128-byte
// swizzled rows), one thread issues tcgen05.mma into one of two accumulators in
// tensor memory, four or eight warps take the finished one through the epilogue
// while the next tile accumulates.  What the operands look like is in the
// descriptors alone:
//   forward            A, B stored with the contraction last (K-major)
//   input gradient     dx = dz W: W is stored [contraction][columns], MN-major
//   weight gradient    dW = dz^T x: both MN-major, contraction = token rows
// With few tokens the operands change sides (kSwap): the weights fill the 128
// rows of the tensor core's tile and the tokens its 16..128 columns, so that no
// row of the machine multiplies padding and the weights are read once.
//
// Long contractions with few tiles are split over the CTAs of a cluster: each
// leaves its partial tile in its own shared memory, and each sums a share of the
// columns over the cluster in rank order (fixed, so results do not vary), with
// no workspace, no counters and nothing to clear.
//
// Experts: the row ranges are read on the device (no host sync).  A row block
// ends at its expert's last row by not storing the rows behind it; a weight
// gradient's last 64 rows are cut to the expert's by zeroing what TMA brought in
// of the next one's in shared memory (in both operands: 0 * NaN would stay), by a
// warp of its own: done by the issuing warp it took 1000 cycles of each tile.
//
// f32 results: the tensor core adds to its f32 accumulator by truncation, an
// error that grows with the length of the sum (measured relative to the norm:
// 4.7e-7 at K = 512, 9e-6 at 8192, 3.8e-5 at 32768).  Behind a 16-bit rounding
// (4e-3 / 5e-4) that is nothing; f32 results are summed in registers, rounded to
// nearest, from accumulators of kSegment * 64 = 512 products each.
#include "launch_cache.h"
#include "linear_common.cuh"

namespace wave {

__device__ int g_linear_status[4]; // [0] code, [1] linear block, [2] role, [3] detail

namespace {

using namespace linear_detail;

constexpr int kTileP = 128;
constexpr int kBK = 64;
constexpr int kChunkBytes = 64 * 128; // 64 rows of 128 bytes: a 64-element MN chunk of a stage
constexpr int kABytes = kTileP * kBK * 2;
constexpr int kMaxStages = 12;
constexpr int kMinStages = 3;
constexpr int kSegment = 8; // stages of an accumulator that is summed in registers
constexpr int kTableBytes = linear_table_bytes(kRaggedRows, kLinearMaxGroups);
constexpr int kSmemLimit = 227 * 1024;

struct Shared {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t tfull[2];
  uint64_t tempty[2];
  // The stage with an expert's last rows: it lands on a barrier of its own (the
  // cutting warp sees only these stages, and a wait for a parity must not skip a
  // turn), and has been cut.
  uint64_t landed[kMaxStages], cut[kMaxStages];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(Shared) <= 1024, "Shared outgrew its slot");

template <int TN, bool kF32> struct Cfg {
  static constexpr int kEpiWarps = TN >= 128 ? 8 : 4;
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kThreadsCut = kThreads + 32; // the weight gradient has a warp that cuts
  static constexpr int kBBytes = TN * kBK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kSlots = kEpiWarps * kSlotBytes;
  // Stages that fit beside a table of so many bytes.
  static constexpr int stages(int table) {
    const int fit = (kSmemLimit - kSmemFixed - table) / kStageBytes;
    return fit < kMaxStages ? fit : kMaxStages;
  }
  static constexpr int kTmemCols = 2 * TN < 32 ? 32 : 2 * TN;
  static constexpr int kSmemFixed = 1024 + 1024 + kSlots; // + the stages, the group table
  static_assert((kSmemLimit - kSmemFixed - kTableBytes) / kStageBytes >= kMinStages, "ring too short");
  static_assert(TN * kTileP * 4 <= kMinStages * kStageBytes, "a partial tile must fit the shortest ring");
};

__device__ __noinline__ void report(int code, int role, int detail) {
  if (atomicCAS(&g_linear_status[0], 0, code) == 0) {
    g_linear_status[1] = static_cast<int>(blockIdx.x);
    g_linear_status[2] = role;
    g_linear_status[3] = detail;
  }
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

template <int W> __device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[W]) {
  static_assert(W == 16 || W == 32 || W == 64, "16, 32 or 64 columns");
  uint32_t r[W];
  if constexpr (W == 64) {
    tmem_ld_32x32b_x32(addr, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
    tmem_ld_32x32b_x32(addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
  } else if constexpr (W == 32)
    tmem_ld_32x32b_x32(addr, r);
  else
    tmem_ld_32x32b_x16(addr, r);
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < W; ++i)
    v[i] = __uint_as_float(r[i]);
}

template <int TN, bool kAMn, bool kBMn, bool kSwap, bool kF32>
__global__ void __launch_bounds__(kAMn && kBMn ? Cfg<TN, kF32>::kThreadsCut : Cfg<TN, kF32>::kThreads, 1)
linear_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
              const __grid_constant__ CUtensorMap tm_d, const __grid_constant__ CUtensorMap tm_z,
              const __grid_constant__ LinearParams p) {
  using C = Cfg<TN, kF32>;
  const int num_stages = p.stages;
  constexpr bool kFull = !kAMn && !kBMn; // the forward pass
  constexpr bool kCut = kAMn && kBMn; // the weight gradient: stages may have to be cut at the last row
  constexpr int kColGroups = C::kEpiWarps / 4;
  constexpr int kMyCols = TN / kColGroups; // columns of an epilogue warp
  // Columns of a chunk.  What only stores takes 64 (of 16 bits: rows of 128 bytes;
  // with 32 the fixed cost of a chunk -- fence, store, waits -- and its latencies
  // come twice as often, 1400 cycles each, which bounded short sums); the forward
  // pass has no registers for more than 32 (8192 x 8192 x 2048 with everything:
  // 222 us, 235 with 64).
  constexpr int W = kSwap || kF32 || kFull ? (kMyCols < 32 ? kMyCols : 32) : 64;
  // The groups of four warps take chunks in turn.
  constexpr int kStride = kF32 || kSwap ? W : W * kColGroups;
  static_assert(!kF32 || kMyCols <= 64, "running sums stay in registers");

  extern __shared__ uint8_t smem_raw[];
  uint8_t *tiles = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Shared *sh = reinterpret_cast<Shared *>(tiles + num_stages * C::kStageBytes);
  uint8_t *slots = tiles + num_stages * C::kStageBytes + 1024;
  GroupTable table;
  table.begin = reinterpret_cast<int *>(slots + C::kSlots);
  table.blocks = table.begin + p.groups + 1;
  volatile int *abort_flag = &sh->abort_flag;

  const int warp = warp_uniform(static_cast<int>(threadIdx.x >> 5));
  const int lane = threadIdx.x & 31;
  const int splits = p.splits;
  const int rank = splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int first_tile = splits > 1 ? static_cast<int>(blockIdx.x) / splits : static_cast<int>(blockIdx.x);
  const int tile_step = splits > 1 ? 0x3FFFFFFF : static_cast<int>(gridDim.x); // a cluster has one tile

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_a);
    tma_prefetch_desc(&tm_b);
    for (int s = 0; s < num_stages; ++s) {
      mbar_init(&sh->full[s], 1);
      mbar_init(&sh->empty[s], 1);
      mbar_init(&sh->landed[s], 1);
      mbar_init(&sh->cut[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&sh->tfull[a], 1);
      mbar_init(&sh->tempty[a], C::kEpiWarps);
    }
    sh->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&sh->tmem_base, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = sh->tmem_base;
  // Up to here only this CTA's own state was touched: it may run while the kernel
  // before this one on the stream is finishing.
  start_after_previous(p.beside);
  if (p.ragged != kRaggedNone)
    build_group_table(table, p.offsets, p.groups, p.ragged == kRaggedK ? p.K : (kSwap ? p.Q : p.P),
                      kSwap ? p.tile_q : kTileP);

  EpiWarp epi_warp;
  epi_warp.slot = slots + (warp - 2) * kSlotBytes;
  epi_warp.map_d = &tm_d;
  epi_warp.map_z = &tm_z;
  epi_warp.lane = lane;
  float col_bias = 0.0f; // tokens as columns: the bias of the lane's feature, fetched while the tile accumulates

  // This CTA's share of a tile's stages.
  auto k_blocks = [&](const Tile &w, int &kb0, int &kb1) {
    const int total = (w.k_len + kBK - 1) / kBK;
    kb0 = splits > 1 ? static_cast<int>(static_cast<long long>(total) * rank / splits) : 0;
    kb1 = splits > 1 ? static_cast<int>(static_cast<long long>(total) * (rank + 1) / splits) : total;
  };

  // Whether the last of them holds an expert's last rows and more.
  auto has_cut = [&](const Tile &w, int kb0, int kb1) {
    return kCut && p.ragged == kRaggedK && (w.k_len & (kBK - 1)) != 0 && kb1 > kb0 && kb1 * kBK > w.k_len;
  };

  if (warp == 0) {
    // ------------------------------------------------------------- loads
    // Like the issuing warp below, the whole warp walks and waits and one elected
    // lane acts: with the loop in one lane's branch the compiler cannot keep the
    // operands of the copies and products in uniform registers, and a stage takes
    // 0.28 us to issue whatever the size of its tile (now 0.18).
    TileWalk<kSwap> walk(p, table, kTileP);
    Tile w;
    Ring ring;
    bool ok = true;
    const bool chosen = elect_one();
    const uint32_t tx = kABytes + static_cast<uint32_t>(p.tile_q) * kBK * 2;
    for (int id = first_tile; ok && walk.get_uniform(id, w); id += tile_step) {
      int kb0, kb1;
      k_blocks(w, kb0, kb1);
      const int za = p.group_a ? w.group : 0, zb = p.group_b ? w.group : 0;
      bool seen = false;
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = warp_wait(&sh->empty[ring.stage], ring.phase ^ 1, abort_flag, seen);
        if (!ok) {
          report(kStatusWaitTimeout, 0, ring.stage);
          break;
        }
        uint8_t *a_dst = tiles + ring.stage * C::kStageBytes;
        uint8_t *b_dst = a_dst + kABytes;
        uint64_t *bar = kCut && kb + 1 == kb1 && has_cut(w, kb0, kb1) ? &sh->landed[ring.stage] : &sh->full[ring.stage];
        const int k = w.k_begin + kb * kBK;
        ring.advance(num_stages);
        seen = warp_peek(&sh->empty[ring.stage], ring.phase ^ 1);
        if (chosen) {
          mbar_arrive_expect_tx(bar, tx);
          if constexpr (kAMn) {
            if (p.chunks_a) {
              tma_load_chunks(a_dst, &tm_a, bar, k, w.p0 / 64, za);
            } else {
#pragma unroll
              for (int c = 0; c < kTileP / 64; ++c)
                tma_load_3d(a_dst + c * kChunkBytes, &tm_a, bar, w.p0 + c * 64, k, za);
            }
          } else {
            tma_load_3d(a_dst, &tm_a, bar, k, w.p0, za);
          }
          if constexpr (kBMn) {
            if (p.chunks_b) {
              tma_load_chunks(b_dst, &tm_b, bar, k, w.q0 / 64, zb);
            } else {
#pragma unroll
              for (int c = 0; c < TN / 64; ++c)
                if (c * 64 < p.tile_q)
                  tma_load_3d(b_dst + c * kChunkBytes, &tm_b, bar, w.q0 + c * 64, k, zb);
            }
          } else {
            tma_load_3d(b_dst, &tm_b, bar, k, w.q0, zb);
          }
        }
        __syncwarp();
      }
    }
    if (!ok)
      bounded_delay(1 << 21); // let copies in flight land before teardown
  } else if (warp == 1) {
    // -------------------------------------------------------- UMMA issue
    // The loop over whole stages holds nothing but a wait, four products and a
    // commit (descriptors are one addition away from those of stage 0).
    const uint32_t idesc = umma_idesc_f16(kTileP, p.tile_q, p.is_bf16, kAMn ? 1 : 0, kBMn ? 1 : 0);
    constexpr uint64_t kStepA = kAMn ? (16 * 128) >> 4 : 2, kStepB = kBMn ? (16 * 128) >> 4 : 2;
    constexpr uint64_t kStep = C::kStageBytes >> 4;
    const uint32_t a_addr = smem_u32(tiles), b_addr = a_addr + kABytes;
    const uint64_t da0 = kAMn ? umma_desc_mnmajor_sw128(a_addr, kChunkBytes, 1024) : umma_desc_kmajor_sw128(a_addr);
    const uint64_t db0 = kBMn ? umma_desc_mnmajor_sw128(b_addr, kChunkBytes, 1024) : umma_desc_kmajor_sw128(b_addr);
    const uint32_t tmem_d = static_cast<uint32_t>(warp_uniform(static_cast<int>(tmem_base)));
    const bool chosen = elect_one();
    TileWalk<kSwap> walk(p, table, kTileP);
    Tile w, next_w;
    Ring ring;
    int acc = 0;
    uint32_t acc_phase = 0, cut_phases = 0; // of cut: a bit to a stage
    bool ok = true;
    bool more_tiles = walk.get_uniform(first_tile, next_w);
    for (int id = first_tile; ok && more_tiles;) {
      w = next_w;
      id += tile_step;
      bool looked = false; // where the next tile lies: worked out while products are under way
      int kb0, kb1;
      k_blocks(w, kb0, kb1);
      const int live = w.k_len & (kBK - 1);
      const bool cut = has_cut(w, kb0, kb1);
      for (int kb = kb0; ok && kb < kb1;) {
        const int end = kF32 ? min(kb + kSegment, kb1) : kb1;
        const bool cut_here = cut && end == kb1;
        const int whole = end - kb - (cut_here ? 1 : 0);
        const uint32_t d = tmem_d + static_cast<uint32_t>(acc * TN);
        ok = warp_wait(&sh->tempty[acc], acc_phase ^ 1, abort_flag, false);
        if (!ok) {
          report(kStatusWaitTimeout, 1, 100 + acc);
          break;
        }
        uint32_t more = 0; // the accumulator holds something
        bool seen = false;
        for (int i = 0; i < whole; ++i) {
          ok = warp_wait(&sh->full[ring.stage], ring.phase, abort_flag, seen);
          if (!ok)
            break;
          tc_fence_after_sync();
          const uint64_t da = da0 + static_cast<uint64_t>(ring.stage) * kStep, db = db0 + static_cast<uint64_t>(ring.stage) * kStep;
          uint64_t *done = &sh->empty[ring.stage];
          ring.advance(num_stages);
          seen = warp_peek(&sh->full[ring.stage], ring.phase);
          if (chosen) {
            umma_ss(d, da, db, idesc, more);
#pragma unroll
            for (int k = 1; k < kBK / 16; ++k)
              umma_ss(d, da + k * kStepA, db + k * kStepB, idesc, 1u);
            umma_commit(done);
          }
          __syncwarp();
          more = 1;
          if (!looked) {
            more_tiles = walk.get_uniform(id, next_w);
            looked = true;
          }
        }
        if constexpr (kCut) {
          if (ok && cut_here) {
            const uint32_t parity = (cut_phases >> ring.stage) & 1u;
            cut_phases ^= 1u << ring.stage;
            ok = warp_wait(&sh->cut[ring.stage], parity, abort_flag, false);
            if (ok) {
              const int steps = (live + 15) / 16;
              tc_fence_after_sync();
              if (chosen) {
                mbar_arrive(&sh->full[ring.stage]); // the stage's turn of this barrier
                const uint64_t da = da0 + static_cast<uint64_t>(ring.stage) * kStep, db = db0 + static_cast<uint64_t>(ring.stage) * kStep;
                for (int k = 0; k < steps; ++k, more = 1)
                  umma_ss(d, da + k * kStepA, db + k * kStepB, idesc, more);
                umma_commit(&sh->empty[ring.stage]);
              }
              __syncwarp();
              ring.advance(num_stages);
            }
          }
        }
        if (!ok) {
          report(kStatusWaitTimeout, 1, ring.stage);
          break;
        }
        if (chosen)
          umma_commit(&sh->tfull[acc]);
        __syncwarp();
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
        kb = end;
      }
      if (ok && !looked)
        more_tiles = walk.get_uniform(id, next_w);
    }
  } else if (kCut && warp == 2 + C::kEpiWarps) {
    // ------------------------------------------------- cutting of last stages
    // Rows [live, the next multiple of 16) of an expert's last stage belong to the
    // next expert or to nobody: zero in both operands before they are multiplied.
    if constexpr (kCut) {
      TileWalk<kSwap> walk(p, table, kTileP);
      Tile w;
      Ring ring;
      uint32_t phases = 0; // of landed: a bit to a stage
      for (int id = first_tile; p.ragged == kRaggedK && walk.get_uniform(id, w); id += tile_step) {
        int kb0, kb1;
        k_blocks(w, kb0, kb1);
        const bool cut = has_cut(w, kb0, kb1);
        ring.stage = (ring.stage + kb1 - kb0 - (cut ? 1 : 0)) % num_stages;
        if (!cut)
          continue;
        const uint32_t parity = (phases >> ring.stage) & 1u;
        phases ^= 1u << ring.stage;
        if (!warp_wait(&sh->landed[ring.stage], parity, abort_flag, false)) {
          report(kStatusWaitTimeout, 3, ring.stage);
          break;
        }
        uint8_t *a_tile = tiles + ring.stage * C::kStageBytes;
        const int live = w.k_len & (kBK - 1), steps = (live + 15) / 16;
        const int vecs = (steps * 16 - live) * 8; // 16-byte pieces in a chunk
        const int chunks = kTileP / 64 + p.tile_q / 64;
        for (int c = 0; c < chunks; ++c)
          for (int i = lane; i < vecs; i += 32)
            *reinterpret_cast<uint4 *>(a_tile + c * kChunkBytes + live * 128 + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&sh->cut[ring.stage]);
        __syncwarp();
        ring.stage = (ring.stage + 1) % num_stages;
      }
    }
  } else {
    // ---------------------------------------------------------- epilogue
    const int quarter = warp & 3; // tensor-memory lanes this warp may read
    const int col0 = ((warp - 2) >> 2) * (kF32 || kSwap ? kMyCols : W);
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    EpiWarp ew = epi_warp;
    TileWalk<kSwap> walk(p, table, kTileP);
    Tile w;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    auto wait_acc = [&]() {
      if (!mbar_wait(&sh->tfull[acc], acc_phase, abort_flag)) {
        if (lane == 0)
          report(kStatusWaitTimeout, 2, 200 + acc);
        return false;
      }
      tc_fence_after_sync();
      return true;
    };
    auto release_acc = [&]() {
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&sh->tempty[acc]);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    };
    // (where the next tile lies is worked out while this one's accumulator is waited for)
    Tile next_w;
    bool more_tiles = walk.get(first_tile, next_w);
    for (int id = first_tile; ok && more_tiles;) {
      w = next_w;
      id += tile_step;
      more_tiles = walk.get(id, next_w);
      int kb0, kb1;
      k_blocks(w, kb0, kb1);
      EpiTile t;
      t.group = w.group;
      t.lane0 = w.p0 + quarter * 32;
      t.lane_end = w.p_end;
      t.q_end = min(w.q_end, w.q0 + p.tile_q);
      if constexpr (kSwap)
        col_bias = column_bias(p, t, lane);
      // columns of this warp that exist, in chunks of W
      const int my_cols = kF32 || kSwap ? min(kMyCols, p.tile_q - col0) : p.tile_q - col0;
      // split: four columns c .. c + 3 of a row side by side, 128 rows of them one after the other
      float4 *part = reinterpret_cast<float4 *>(tiles) + quarter * 32 + lane;
      auto chunk = [&](int c, float (&v)[W], const Ahead<W> &f) {
        if (splits > 1) {
#pragma unroll
          for (int j = 0; j < W; j += 4)
            part[(c + j) / 4 * kTileP] = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        } else if constexpr (kSwap) {
          epilogue_columns<kF32, W>(p, t, w.q0 + c, v, col_bias, ew.slot, lane);
        } else {
          epilogue_rows<kF32, W, kFull>(p, t, w.q0 + c, v, f, ew);
        }
      };
      if constexpr (kF32) {
        float run[kMyCols];
#pragma unroll
        for (int j = 0; j < kMyCols; ++j)
          run[j] = 0.0f;
        for (int kb = kb0; kb < kb1 && ok; kb += kSegment) {
          ok = wait_acc();
          if (!ok)
            break;
#pragma unroll
          for (int c = 0; c < kMyCols; c += W) {
            if (c >= my_cols)
              break;
            float v[W];
            tmem_load<W>(lane_addr + static_cast<uint32_t>(acc * TN + col0 + c), v);
#pragma unroll
            for (int j = 0; j < W; ++j)
              run[c + j] += v[j];
          }
          release_acc();
        }
        if (!ok)
          break;
#pragma unroll
        for (int c = 0; c < kMyCols; c += W) {
          if (c >= my_cols)
            break;
          Ahead<W> f;
          if (!kSwap && kFull && splits == 1)
            fetch_ahead<W>(f, p, t, w.q0 + col0 + c, lane);
          float v[W];
#pragma unroll
          for (int j = 0; j < W; ++j)
            v[j] = run[c + j];
          chunk(col0 + c, v, f);
        }
      } else {
        const bool empty = kb0 == kb1; // nothing to multiply: the epilogue of zero
        Ahead<W> next;
        if (!kSwap && kFull && splits == 1 && my_cols > 0)
          fetch_ahead<W>(next, p, t, w.q0 + col0, lane);
        if (!empty && !wait_acc()) {
          ok = false;
          break;
        }
#pragma unroll 1
        for (int c = 0; c < my_cols; c += kStride) {
          float v[W];
          if (empty) {
#pragma unroll
            for (int j = 0; j < W; ++j)
              v[j] = 0.0f;
          } else {
            tmem_load<W>(lane_addr + static_cast<uint32_t>(acc * TN + col0 + c), v);
          }
          if (!empty && c + kStride >= my_cols)
            release_acc(); // read out: the tile after the next may use it
          chunk(col0 + c, v, next);
          if (!kSwap && kFull && splits == 1 && c + kStride < my_cols)
            fetch_ahead<W>(next, p, t, w.q0 + col0 + c + kStride, lane);
        }
        if (!empty && my_cols <= 0)
          release_acc();
      }
    }
    if (lane == 0)
      tma_store_wait<0>(); // the slots outlive the stores that read them
    if (p.zero_rest && p.ragged == kRaggedRows) {
      // the rows in front of the first and behind the last group
      const int rows = kSwap ? p.Q : p.P, cols = kSwap ? p.P : p.Q;
      const int wid = static_cast<int>(blockIdx.x) * C::kEpiWarps + warp - 2, warps = static_cast<int>(gridDim.x) * C::kEpiWarps;
      zero_rows(p.D, kF32 ? 4 : 2, p.ldd, 0, table.begin[0], cols, wid, warps, lane);
      zero_rows(p.D, kF32 ? 4 : 2, p.ldd, table.begin[p.groups], rows, cols, wid, warps, lane);
      if (p.Z) {
        zero_rows(p.Z, 2, p.ldz, 0, table.begin[0], cols, wid, warps, lane);
        zero_rows(p.Z, 2, p.ldz, table.begin[p.groups], rows, cols, wid, warps, lane);
      }
    }
  }

  if (splits > 1) {
    // The partial tiles of the cluster: each CTA takes columns of all 128 rows
    // and adds the parts in rank order.  Every CTA of the cluster passes both
    // barriers whatever happened above.
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    if (warp >= 2 && warp < 2 + C::kEpiWarps && *abort_flag == 0) {
      const int quarter = warp & 3, half = (warp - 2) >> 2;
      EpiWarp ew = epi_warp;
      TileWalk<kSwap> walk(p, table, kTileP);
      Tile w;
      if (walk.get(first_tile, w)) {
        EpiTile t;
        t.group = w.group;
        t.lane0 = w.p0 + quarter * 32;
        t.lane_end = w.p_end;
        t.q_end = min(w.q_end, w.q0 + p.tile_q);
        uint32_t peer[kLinearMaxSplits];
#pragma unroll
        for (int s = 0; s < kLinearMaxSplits; ++s)
          peer[s] = s < splits ? map_to_cta(tiles, static_cast<uint32_t>(s)) + (quarter * 32 + lane) * 16 : 0u;
        // four columns from all parts, in flight together, added in rank order
        auto four = [&](int col) {
          float4 part[kLinearMaxSplits];
#pragma unroll
          for (int s = 0; s < kLinearMaxSplits; ++s)
            if (s < splits)
              part[s] = ld_cluster_f32x4(peer[s] + col / 4 * (kTileP * 16));
          float4 sum = part[0];
#pragma unroll
          for (int s = 1; s < kLinearMaxSplits; ++s)
            if (s < splits) {
              sum.x += part[s].x;
              sum.y += part[s].y;
              sum.z += part[s].z;
              sum.w += part[s].w;
            }
          return sum;
        };
        if constexpr (kSwap) {
          // four tokens at a time
          const int live = t.q_end - w.q0;
          for (int i = rank + half * splits; i * 4 < live; i += kColGroups * splits) {
            const float4 f = four(i * 4);
            float v[4] = {f.x, f.y, f.z, f.w};
            epilogue_columns<kF32, 4>(p, t, w.q0 + i * 4, v, col_bias, ew.slot, lane);
          }
        } else {
          constexpr int V = 16; // columns at a time
          for (int i = rank + half * splits; i * V < p.tile_q; i += kColGroups * splits) {
            const int q0 = w.q0 + i * V;
            Ahead<V> f;
            if constexpr (kFull)
              fetch_ahead<V>(f, p, t, q0, lane);
            float v[V];
#pragma unroll
            for (int j = 0; j < V; j += 4) {
              const float4 q = four(i * V + j);
              v[j] = q.x;
              v[j + 1] = q.y;
              v[j + 2] = q.z;
              v[j + 3] = q.w;
            }
            epilogue_rows<kF32, V, kFull>(p, t, q0, v, f, ew);
          }
        }
      }
    }
    if (warp >= 2 && lane == 0)
      tma_store_wait<0>();
    __syncwarp();
    cluster_arrive(); // nobody leaves while its part may still be read
    cluster_wait();
  }

  end_after_previous(p.beside);
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

template <int TN, bool kAMn, bool kBMn, bool kSwap, bool kF32>
cudaError_t launch_one(const LinearMaps &m, const LinearParams &p, const LinearLaunch &l,
                       cudaStream_t stream) {
  using C = Cfg<TN, kF32>;
  if (p.stages < kMinStages || p.stages > C::stages(linear_table_bytes(p.ragged, p.groups)))
    return cudaErrorInvalidValue;
  auto kernel = linear_kernel<TN, kAMn, kBMn, kSwap, kF32>;
  cudaError_t err = prepare_kernel(kernel, kSmemLimit, nullptr);
  if (err != cudaSuccess)
    return err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(l.grid));
  cfg.blockDim = dim3(kAMn && kBMn ? C::kThreadsCut : C::kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(C::kSmemFixed) + static_cast<size_t>(p.stages) * C::kStageBytes + linear_table_bytes(p.ragged, p.groups);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.numAttrs = 0;
  if (l.pdl) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.splits > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = static_cast<unsigned>(p.splits);
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kernel, m.a, m.b, m.d, m.z, p);
}

template <bool kAMn, bool kBMn, bool kSwap, bool kF32>
cudaError_t launch_tile(const LinearMaps &m, const LinearParams &p, const LinearLaunch &l,
                        cudaStream_t stream) {
  if constexpr (kSwap) {
    switch (l.tile_n) {
    case 16:
      return launch_one<16, kAMn, kBMn, kSwap, kF32>(m, p, l, stream);
    case 32:
      return launch_one<32, kAMn, kBMn, kSwap, kF32>(m, p, l, stream);
    }
  }
  switch (l.tile_n) {
  case 64:
    return launch_one<64, kAMn, kBMn, kSwap, kF32>(m, p, l, stream);
  case 128:
    return launch_one<128, kAMn, kBMn, kSwap, kF32>(m, p, l, stream);
  }
  if constexpr (!kSwap && !kF32) {
    if (l.tile_n == 256)
      return launch_one<256, kAMn, kBMn, kSwap, kF32>(m, p, l, stream);
  }
  return cudaErrorInvalidValue;
}

template <bool kF32>
cudaError_t launch_layout(const LinearMaps &m, const LinearParams &p, const LinearLaunch &l,
                          cudaStream_t stream) {
  if (!l.a_mn && !l.b_mn)
    return l.swap ? launch_tile<false, false, true, kF32>(m, p, l, stream)
                  : launch_tile<false, false, false, kF32>(m, p, l, stream);
  if (l.swap)
    return cudaErrorInvalidValue;
  if (!l.a_mn && l.b_mn) {
    if constexpr (!kF32) // the input gradient has the operands' type
      return launch_tile<false, true, false, kF32>(m, p, l, stream);
  }
  if (l.a_mn && l.b_mn)
    return launch_tile<true, true, false, kF32>(m, p, l, stream);
  return cudaErrorInvalidValue;
}

} // namespace

int linear_max_stages(int tile_n, int out_f32, int ragged, int groups) {
  const int table = linear_table_bytes(ragged, groups);
  switch (tile_n) {
  case 16: return out_f32 ? Cfg<16, true>::stages(table) : Cfg<16, false>::stages(table);
  case 32: return out_f32 ? Cfg<32, true>::stages(table) : Cfg<32, false>::stages(table);
  case 64: return out_f32 ? Cfg<64, true>::stages(table) : Cfg<64, false>::stages(table);
  case 128: return out_f32 ? Cfg<128, true>::stages(table) : Cfg<128, false>::stages(table);
  }
  return Cfg<256, false>::stages(table);
}

cudaError_t launch_linear(const LinearMaps &m, const LinearParams &p, const LinearLaunch &l, cudaStream_t stream) {
  if (l.pair)
    return launch_linear_pair(m, p, l, stream);
  return l.out_f32 ? launch_layout<true>(m, p, l, stream) : launch_layout<false>(m, p, l, stream);
}

cudaError_t linear_read_status(int out[4], bool clear) {
  cudaError_t err = cudaMemcpyFromSymbol(out, g_linear_status, sizeof(int) * 4);
  if (err == cudaSuccess && clear) {
    int zero[4] = {0, 0, 0, 0};
    err = cudaMemcpyToSymbol(g_linear_status, zero, sizeof(zero));
  }
  return err;
}

} // namespace wave
