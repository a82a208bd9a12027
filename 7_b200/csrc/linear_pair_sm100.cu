// Products of the linear layers on CTA pairs, for problems with many tiles: two
// CTAs of a cluster compute one 256 x (up to 256) tile with tcgen05.mma
// cta_group::2.  Each loads its own 128 rows of A and its own half of the tile's
// B (no multicast) and receives its 128 accumulator rows in its own tensor
// memory, so a step of 64 moves 32 KB to a CTA where the one-CTA kernel moves 48
// for the same outputs: a deeper ring and a third less shared-memory traffic.
// Operand layouts, experts and the epilogue are those of linear_sm100.cu.
//
// With experts the sides may change (kSwap): 256 features are the tile's rows, and
// its columns the tokens, so a tile is as wide as it has tokens for (an expert's
// are shared out evenly, in steps of 32), where rows come in whole 256s.  A step's
// time does not fall with the columns alone: what it loads and reads of shared
// memory, 128 rows of A and up to as much of B a CTA, keeps the memory as busy as
// 256 columns keep the tensor cores; so the host also picks the columns that are
// loaded (tile_q).  Rows / columns in us, bf16: 3001 tokens, 1032 x 1544, 32 experts
// 42 / 36; 8192, 4096 x 2048, 16 130 / 122; 16384, 2048 x 1024, 64 96 / 87; with
// whole blocks (16384, 8192 x 4096, 8) 771 / 772.
//
// Barriers across the pair:
//   full[s]    in the leader, armed by its loader with the bytes of both CTAs'
//              loads (an arrival of the other CTA's loader for each stage was
//              tried: a remote arrival with release costs that thread so long that
//              8192^3 took 1500 us)
//   landed[s]  one per CTA: the last stage of an expert's weight gradient lands
//              here, and the CTA's cutting warp zeroes the rows behind the expert's
//              last (several such stages may be in the ring, so each has a barrier)
//   cut[s]     in the leader: both CTAs have done so; the leader's issuing warp
//              then completes full[s] itself
//   empty[s], tfull[a]  one per CTA; the leader's tcgen05.commit arrives on both
//   tempty[a]  in the leader; the epilogue warps of both CTAs arrive
#include "launch_cache.h"
#include "linear_common.cuh"

namespace wave {

__device__ int g_linear_pair_status[4]; // [0] code, [1] linear block, [2] role, [3] detail

namespace {

using namespace linear_detail;

constexpr int kRows = 128; // rows of A, and of the accumulator, in each CTA
constexpr int kPairP = 256;
constexpr int kTN = 256;
constexpr int kBK = 64;
constexpr int kChunkBytes = 64 * 128;
constexpr int kABytes = kRows * kBK * 2;
constexpr int kBBytes = kTN / 2 * kBK * 2;
constexpr int kStageBytes = kABytes + kBBytes;
constexpr int kMaxStages = 6; // five where the experts' table is long
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kThreadsCut = kThreads + 32; // the weight gradient has a warp that cuts
constexpr int kSlots = kEpiWarps * kSlotBytes;
constexpr int kSmemLimit = 227 * 1024;
constexpr int kSmemFixed = 1024 + 1024 + kSlots; // + the stages, the group table
static_assert(kSmemFixed + 5 * kStageBytes + linear_table_bytes(kRaggedRows, kLinearMaxGroups) <= kSmemLimit,
              "does not fit the shared memory of an SM");

struct PairShared {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t tfull[2];
  uint64_t tempty[2];
  uint64_t landed[kMaxStages];
  uint64_t cut[kMaxStages];
  uint32_t tmem_base;
  int abort_flag;
};

__device__ __noinline__ void pair_report(int code, int role, int detail) {
  if (atomicCAS(&g_linear_pair_status[0], 0, code) == 0) {
    g_linear_pair_status[1] = static_cast<int>(blockIdx.x);
    g_linear_pair_status[2] = role;
    g_linear_pair_status[3] = detail;
  }
}

__device__ __forceinline__ void tma_load_3d_pair(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
               " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar) & kPeerBitMask), "r"(x), "r"(y), "r"(z)
               : "memory");
}

__device__ __forceinline__ void tma_load_chunks_pair(void *dst, const CUtensorMap *map, uint64_t *bar, int row, int chunk, int z) {
  asm volatile("cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
               " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar) & kPeerBitMask), "r"(0), "r"(row), "r"(chunk), "r"(z)
               : "memory");
}

template <bool kAMn, bool kBMn, bool kSwap>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kAMn && kBMn ? kThreadsCut : kThreads, 1)
linear_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                   const __grid_constant__ CUtensorMap tm_d, const __grid_constant__ CUtensorMap tm_z,
                   const __grid_constant__ LinearParams p) {
  constexpr bool kFull = !kAMn && !kBMn && !kSwap; // the forward pass, tokens as rows
  constexpr int kW = kFull || kSwap ? 32 : 64; // columns of an epilogue chunk (see linear_sm100.cu); the two groups of four warps take turns
  constexpr bool kCut = kAMn && kBMn;
  const int num_stages = p.stages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *tiles = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  PairShared *sh = reinterpret_cast<PairShared *>(tiles + num_stages * kStageBytes);
  uint8_t *slots = tiles + num_stages * kStageBytes + 1024;
  GroupTable table;
  table.begin = reinterpret_cast<int *>(slots + kSlots);
  table.blocks = table.begin + p.groups + 1;
  volatile int *abort_flag = &sh->abort_flag;

  const int warp = warp_uniform(static_cast<int>(threadIdx.x >> 5));
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const bool leader = rank == 0;
  const int first_tile = static_cast<int>(blockIdx.x >> 1), tile_step = static_cast<int>(gridDim.x >> 1);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_a);
    tma_prefetch_desc(&tm_b);
    for (int s = 0; s < num_stages; ++s) {
      mbar_init(&sh->full[s], 1);
      mbar_init(&sh->empty[s], 1);
      mbar_init(&sh->landed[s], 1);
      mbar_init(&sh->cut[s], 2);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&sh->tfull[a], 1);
      mbar_init(&sh->tempty[a], 2 * kEpiWarps);
    }
    sh->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(&sh->tmem_base, 2 * kTN);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_arrive(); // the peer's barriers must be there before anything signals them
  cluster_wait();
  tc_fence_after_sync();
  const uint32_t tmem_base = sh->tmem_base;
  start_after_previous(p.beside);
  if (p.ragged != kRaggedNone)
    build_group_table(table, p.offsets, p.groups, p.ragged == kRaggedK ? p.K : (kSwap ? p.Q : p.P), kSwap ? p.tile_q : kPairP);

  // Contraction indices of stage kb, and whether rows behind them have to be cut away.
  auto live_of = [](const Tile &w, int kb) { return min(kBK, w.k_len - kb * kBK); };
  auto is_cut = [&](int live) { return kCut && p.ragged == kRaggedK && live < kBK; };
  // The stage that has to be cut is the first of its tile in the ring, and its
  // products follow those of the next kCutLag, so that the cutting is not waited for
  // (15 experts of 546 rows, 4096 x 2048: the last in both 141 us; after 1 / 2 / 3
  // others 127 / 127.5 / 126.5, of 1010 rows 208, 196 / 199 / 196).
  constexpr int kCutLag = 1;

  if (warp == 0) {
    // ------------------------------------------------------------- loads
    TileWalk<kSwap, kSwap> walk(p, table, kPairP);
    Tile w;
    Ring ring;
    bool ok = true;
    const bool chosen = elect_one();
    const int half_q = p.tile_q / 2;
    const uint32_t tx = kABytes + static_cast<uint32_t>(half_q) * kBK * 2; // one CTA's bytes
    for (int id = first_tile; ok && walk.get_uniform(id, w); id += tile_step) {
      const int kbs = (w.k_len + kBK - 1) / kBK;
      const int za = p.group_a ? w.group : 0, zb = p.group_b ? w.group : 0;
      const int pa = w.p0 + rank * kRows, qb = w.q0 + rank * (kSwap ? w.n / 2 : half_q);
      bool seen = false;
      const bool cut = is_cut(live_of(w, kbs - 1));
      for (int i = 0; i < kbs; ++i) {
        const int kb = !cut ? i : i == 0 ? kbs - 1 : i - 1;
        ok = warp_wait(&sh->empty[ring.stage], ring.phase ^ 1, abort_flag, seen);
        if (!ok) {
          pair_report(kStatusWaitTimeout, 0, ring.stage);
          break;
        }
        uint8_t *a_dst = tiles + ring.stage * kStageBytes;
        uint8_t *b_dst = a_dst + kABytes;
        uint64_t *bar = &sh->full[ring.stage];
        uint64_t *landed = &sh->landed[ring.stage];
        const int k = w.k_begin + kb * kBK;
        ring.advance(num_stages);
        seen = warp_peek(&sh->empty[ring.stage], ring.phase ^ 1);
        if (kCut && cut && i == 0) {
          if (chosen) {
            // this CTA's bytes on its own barrier: the cutting warp takes them over
            mbar_arrive_expect_tx(landed, tx);
            if (p.chunks_a) {
              tma_load_chunks(a_dst, &tm_a, landed, k, pa / 64, za);
            } else {
              for (int c = 0; c < kRows / 64; ++c)
                tma_load_3d(a_dst + c * kChunkBytes, &tm_a, landed, pa + c * 64, k, za);
            }
            if (p.chunks_b) {
              tma_load_chunks(b_dst, &tm_b, landed, k, qb / 64, zb);
            } else {
              for (int c = 0; c < half_q / 64; ++c)
                tma_load_3d(b_dst + c * kChunkBytes, &tm_b, landed, qb + c * 64, k, zb);
            }
          }
        } else if (chosen) {
          if (leader)
            mbar_arrive_expect_tx(bar, 2 * tx);
          if constexpr (kAMn) {
            if (p.chunks_a) {
              tma_load_chunks_pair(a_dst, &tm_a, bar, k, pa / 64, za);
            } else {
#pragma unroll
              for (int c = 0; c < kRows / 64; ++c)
                tma_load_3d_pair(a_dst + c * kChunkBytes, &tm_a, bar, pa + c * 64, k, za);
            }
          } else {
            tma_load_3d_pair(a_dst, &tm_a, bar, k, pa, za);
          }
          if constexpr (kBMn) {
            if (p.chunks_b) {
              tma_load_chunks_pair(b_dst, &tm_b, bar, k, qb / 64, zb);
            } else {
#pragma unroll
              for (int c = 0; c < kTN / 128; ++c)
                if (c * 64 < half_q)
                  tma_load_3d_pair(b_dst + c * kChunkBytes, &tm_b, bar, qb + c * 64, k, zb);
            }
          } else {
            tma_load_3d_pair(b_dst, &tm_b, bar, k, qb, zb);
          }
        }
        __syncwarp();
      }
    }
    if (!ok)
      bounded_delay(1 << 21);
  } else if (warp == 1) {
    // ------------------------------------------------ UMMA issue (leader)
    if (leader) {
      uint32_t idesc = umma_idesc_f16(kPairP, p.tile_q, p.is_bf16, kAMn ? 1 : 0, kBMn ? 1 : 0);
      constexpr uint64_t kStepA = kAMn ? (16 * 128) >> 4 : 2, kStepB = kBMn ? (16 * 128) >> 4 : 2;
      constexpr uint64_t kStep = kStageBytes >> 4;
      const uint32_t a_addr = smem_u32(tiles), b_addr = a_addr + kABytes;
      const uint64_t da0 = kAMn ? umma_desc_mnmajor_sw128(a_addr, kChunkBytes, 1024) : umma_desc_kmajor_sw128(a_addr);
      const uint64_t db0 = kBMn ? umma_desc_mnmajor_sw128(b_addr, kChunkBytes, 1024) : umma_desc_kmajor_sw128(b_addr);
      const uint32_t tmem_d = static_cast<uint32_t>(warp_uniform(static_cast<int>(tmem_base)));
      const bool chosen = elect_one();
      TileWalk<kSwap, kSwap> walk(p, table, kPairP);
      Tile w, next_w;
      Ring ring;
      int acc = 0;
      uint32_t acc_phase = 0, cut_phases = 0; // of cut: a bit to a stage
      bool ok = true;
      bool more_tiles = walk.get_uniform(first_tile, next_w);
      for (int id = first_tile; ok && more_tiles;) {
        w = next_w;
        if constexpr (kSwap)
          idesc = umma_idesc_f16(kPairP, w.n, p.is_bf16, kAMn ? 1 : 0, kBMn ? 1 : 0);
        id += tile_step;
        bool looked = false; // where the next tile lies: worked out while products are under way
        const int kbs = (w.k_len + kBK - 1) / kBK;
        if (kbs > 0) {
          const int live = live_of(w, kbs - 1);
          const bool cut = is_cut(live);
          const int whole = kbs - (cut ? 1 : 0);
          const uint32_t d = tmem_d + static_cast<uint32_t>(acc * kTN);
          uint32_t more = 0; // the accumulator holds something
          ok = warp_wait(&sh->tempty[acc], acc_phase ^ 1, abort_flag, false);
          if (!ok) {
            pair_report(kStatusWaitTimeout, 1, 100 + acc);
            break;
          }
          const int cut_stage = ring.stage;
          if (cut)
            ring.advance(num_stages);
          auto issue = [&](int stages) {
            bool seen = false;
            for (int i = 0; i < stages; ++i) {
              ok = warp_wait(&sh->full[ring.stage], ring.phase, abort_flag, seen);
              if (!ok) {
                pair_report(kStatusWaitTimeout, 1, ring.stage);
                break;
              }
              tc_fence_after_sync();
              const uint64_t da = da0 + static_cast<uint64_t>(ring.stage) * kStep, db = db0 + static_cast<uint64_t>(ring.stage) * kStep;
              uint64_t *done = &sh->empty[ring.stage];
              ring.advance(num_stages);
              seen = warp_peek(&sh->full[ring.stage], ring.phase);
              if (chosen) {
                umma_ss_pair(d, da, db, idesc, more);
#pragma unroll
                for (int k = 1; k < kBK / 16; ++k)
                  umma_ss_pair(d, da + k * kStepA, db + k * kStepB, idesc, 1u);
                umma_commit_pair(done, 3); // frees the stage in both CTAs
              }
              __syncwarp();
              more = 1;
              if (!looked) {
                more_tiles = walk.get_uniform(id, next_w);
                looked = true;
              }
            }
          };
          const int before = cut ? min(whole, kCutLag) : whole;
          issue(before);
          if (!ok)
            break;
          if constexpr (kCut) {
            if (cut) {
              const uint32_t parity = (cut_phases >> cut_stage) & 1u;
              cut_phases ^= 1u << cut_stage;
              ok = warp_wait_cluster(&sh->cut[cut_stage], parity, abort_flag);
              if (!ok) {
                pair_report(kStatusWaitTimeout, 1, 70 + cut_stage);
                break;
              }
              fence_proxy_async_smem();
              tc_fence_after_sync();
              const int steps = (live + 15) / 16;
              if (chosen) {
                mbar_arrive(&sh->full[cut_stage]); // the stage's turn of this barrier
                const uint64_t da = da0 + static_cast<uint64_t>(cut_stage) * kStep, db = db0 + static_cast<uint64_t>(cut_stage) * kStep;
                umma_ss_pair(d, da, db, idesc, more);
                for (int k = 1; k < steps; ++k)
                  umma_ss_pair(d, da + k * kStepA, db + k * kStepB, idesc, 1u);
                umma_commit_pair(&sh->empty[cut_stage], 3);
              }
              __syncwarp();
              more = 1;
              issue(whole - before);
              if (!ok)
                break;
            }
          }
          if (chosen)
            umma_commit_pair(&sh->tfull[acc], 3);
          __syncwarp();
          if (++acc == 2) {
            acc = 0;
            acc_phase ^= 1;
          }
        }
        if (!looked)
          more_tiles = walk.get_uniform(id, next_w);
      }
    }
  } else if (kCut && warp == 2 + kEpiWarps) {
    // ------------------------------------- cutting of last stages (both CTAs)
    if constexpr (kCut) {
      TileWalk<kSwap, kSwap> walk(p, table, kPairP);
      Tile w;
      Ring ring;
      uint32_t phases = 0; // of landed: a bit to a stage
      for (int id = first_tile; p.ragged == kRaggedK && walk.get_uniform(id, w); id += tile_step) {
        const int kbs = (w.k_len + kBK - 1) / kBK;
        if (kbs <= 0)
          continue;
        const int live = live_of(w, kbs - 1);
        const bool cut = is_cut(live);
        const int stage = ring.stage;
        ring.stage = (ring.stage + kbs) % num_stages;
        if (!cut)
          continue;
        const uint32_t parity = (phases >> stage) & 1u;
        phases ^= 1u << stage;
        if (!warp_wait(&sh->landed[stage], parity, abort_flag, false)) {
          pair_report(kStatusWaitTimeout, 3, stage);
          break;
        }
        uint8_t *a_tile = tiles + stage * kStageBytes;
        const int steps = (live + 15) / 16;
        const int vecs = (steps * 16 - live) * 8; // 16-byte pieces in a chunk
        const int chunks = kRows / 64 + p.tile_q / 128;
        for (int c = 0; c < chunks; ++c)
          for (int i = lane; i < vecs; i += 32)
            *reinterpret_cast<uint4 *>(a_tile + c * kChunkBytes + live * 128 + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0)
          mbar_arrive_cluster(map_to_cta(&sh->cut[stage], 0));
        __syncwarp();
      }
    }
  } else {
    // ---------------------------------------------------------- epilogue
    const int quarter = warp & 3;
    const int col0 = ((warp - 2) >> 2) * kW;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    EpiWarp ew{slots + (warp - 2) * kSlotBytes, &tm_d, &tm_z, lane};
    const uint32_t tempty_leader[2] = {map_to_cta(&sh->tempty[0], 0), map_to_cta(&sh->tempty[1], 0)};
    TileWalk<kSwap, kSwap> walk(p, table, kPairP);
    Tile w;
    int acc = 0;
    uint32_t acc_phase = 0;
    auto release = [&]() {
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0)
        mbar_arrive_cluster_relaxed(tempty_leader[acc]);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    };
    // (where the next tile lies is worked out while this one's accumulator is waited for)
    Tile next_w;
    bool more_tiles = walk.get(first_tile, next_w);
    for (int id = first_tile; more_tiles;) {
      w = next_w;
      id += tile_step;
      more_tiles = walk.get(id, next_w);
      const bool empty = w.k_len <= 0; // nothing to multiply: the epilogue of zero
      EpiTile t;
      t.group = w.group;
      t.lane0 = w.p0 + rank * kRows + quarter * 32;
      t.lane_end = w.p_end;
      const int cols = kSwap ? w.n : p.tile_q;
      t.q_end = min(w.q_end, w.q0 + cols);
      const int my_cols = cols - col0;
      float col_bias = 0.0f; // tokens as columns: the bias of the lane's feature
      if constexpr (kSwap)
        col_bias = column_bias(p, t, lane);
      Ahead<kW> next;
      if (kFull && my_cols > 0)
        fetch_ahead<kW>(next, p, t, w.q0 + col0, lane);
      if (!empty) {
        if (!mbar_wait(&sh->tfull[acc], acc_phase, abort_flag)) {
          if (lane == 0)
            pair_report(kStatusWaitTimeout, 2, 200 + acc);
          break;
        }
        tc_fence_after_sync();
      }
#pragma unroll 1
      for (int c = 0; c < my_cols; c += 2 * kW) {
        float v[kW];
        if (empty) {
#pragma unroll
          for (int j = 0; j < kW; ++j)
            v[j] = 0.0f;
        } else {
          uint32_t r[kW];
          const uint32_t at = lane_addr + static_cast<uint32_t>(acc * kTN + col0 + c);
          tmem_ld_32x32b_x32(at, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
          if constexpr (kW == 64)
            tmem_ld_32x32b_x32(at + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < kW; ++j)
            v[j] = __uint_as_float(r[j]);
          if (c + 2 * kW >= my_cols)
            release(); // read out: the tile after the next may use it
        }
        if constexpr (kSwap)
          epilogue_columns<false, kW>(p, t, w.q0 + col0 + c, v, col_bias, ew.slot, lane);
        else
          epilogue_rows<false, kW, kFull>(p, t, w.q0 + col0 + c, v, next, ew);
        if (kFull && c + 2 * kW < my_cols)
          fetch_ahead<kW>(next, p, t, w.q0 + col0 + c + 2 * kW, lane);
      }
      if (!empty && my_cols <= 0)
        release();
    }
    if (lane == 0)
      tma_store_wait<0>(); // the slots outlive the stores that read them
    if (p.zero_rest && p.ragged == kRaggedRows) {
      const int wid = static_cast<int>(blockIdx.x) * kEpiWarps + warp - 2, warps = static_cast<int>(gridDim.x) * kEpiWarps;
      const int rows = kSwap ? p.Q : p.P, cols = kSwap ? p.P : p.Q;
      zero_rows(p.D, 2, p.ldd, 0, table.begin[0], cols, wid, warps, lane);
      zero_rows(p.D, 2, p.ldd, table.begin[p.groups], rows, cols, wid, warps, lane);
      if (p.Z) {
        zero_rows(p.Z, 2, p.ldz, 0, table.begin[0], cols, wid, warps, lane);
        zero_rows(p.Z, 2, p.ldz, table.begin[p.groups], rows, cols, wid, warps, lane);
      }
    }
  }

  end_after_previous(p.beside);
  // Neither CTA may leave, or free tensor memory, while its partner can still
  // read its shared memory, signal its barriers or write its accumulator.
  tc_fence_before_sync();
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, 2 * kTN);
  }
}

template <bool kAMn, bool kBMn, bool kSwap>
cudaError_t launch_one(const LinearMaps &m, const LinearParams &p, const LinearLaunch &l, cudaStream_t stream) {
  if (p.stages != linear_pair_stages(p.ragged, p.groups))
    return cudaErrorInvalidValue;
  auto kernel = linear_pair_kernel<kAMn, kBMn, kSwap>;
  cudaError_t err = prepare_kernel(kernel, kSmemLimit, nullptr);
  if (err != cudaSuccess)
    return err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(l.grid));
  cfg.blockDim = dim3(kAMn && kBMn ? kThreadsCut : kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(kSmemFixed) + static_cast<size_t>(p.stages) * kStageBytes +
                         linear_table_bytes(p.ragged, p.groups);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = l.pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, m.a, m.b, m.d, m.z, p);
}

} // namespace

int linear_pair_stages(int ragged, int groups) {
  const int fit = (kSmemLimit - kSmemFixed - linear_table_bytes(ragged, groups)) / kStageBytes;
  return fit < kMaxStages ? fit : kMaxStages;
}

cudaError_t launch_linear_pair(const LinearMaps &m, const LinearParams &p, const LinearLaunch &l, cudaStream_t stream) {
  if (l.swap) { // with experts only
    if (l.b_mn || p.ragged != kRaggedRows)
      return cudaErrorInvalidValue;
    return l.a_mn ? launch_one<true, false, true>(m, p, l, stream) : launch_one<false, false, true>(m, p, l, stream);
  }
  if (!l.a_mn)
    return l.b_mn ? launch_one<false, true, false>(m, p, l, stream) : launch_one<false, false, false>(m, p, l, stream);
  return l.b_mn ? launch_one<true, true, false>(m, p, l, stream) : cudaErrorInvalidValue;
}

cudaError_t linear_pair_read_status(int out[4], bool clear) {
  cudaError_t err = cudaMemcpyFromSymbol(out, g_linear_pair_status, sizeof(int) * 4);
  if (err == cudaSuccess && clear) {
    int zero[4] = {0, 0, 0, 0};
    err = cudaMemcpyToSymbol(g_linear_pair_status, zero, sizeof(zero));
  }
  return err;
}

} // namespace wave
