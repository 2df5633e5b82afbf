// The e4m3 product with power-of-two block scales (see block_matmul.cuh for the arithmetic): the tensor
// core applies the scales itself (tcgen05.mma kind::mxf8f6f4.block_scale), so one 128 x 256 accumulator
// (256 x 256 over a pair of CTAs, kPair) stays in tensor memory for the whole K loop and nothing is
// promoted in registers.
//
// A scale column of tensor memory holds four bytes per lane; they are filled with the scales of four
// consecutive K blocks, and the instruction descriptor of each stage selects its byte, so scales are
// copied to tensor memory once per four stages, from 32 x 16-byte images that a warp builds in shared
// memory (activations: one word of four bytes per row; weights: the exponent of the f32 power of two,
// the same for the 128 rows of a block).
//
// A second accumulator would leave tensor memory no room for the scales.  When a tile is complete the
// epilogue warps drain it into registers, hand tensor memory back and store while the next tile is
// multiplied.
//
// What bounds a large product is power: a pair holds half of the weight rows in each CTA, which costs a
// third less traffic from L2 and shared memory, and the tiles go through the result in bands.
//
// Measured on a B200, 8192 x 4096 x 7168: 163 to 166 us = 2950 TFLOP/s in a short run; back to back under the power
// limit 191 to 194 us = 2480 TFLOP/s at 1250 MHz, as long as a library e4m3 product without block scales (195; one
// CTA to a tile 210, and without bands 218).
#pragma once

#include "block_matmul.cuh"

namespace fmoe {

constexpr int kHwThreads = 384;                   // warps 0-3: TMA, MMA, scale images (two); warps 4-11: epilogue
constexpr int kHwEpiWarps = 8;
constexpr int kHwTileN = 256;
constexpr int kHwEpiBytes = kHwEpiWarps * 32 * kBmmEpiPitch * 4;
constexpr int kHwSfSlots = 4;                     // ring of scale images, four K blocks a slot
constexpr int kHwSfSlotBytes = 512 + 2 * 512;     // activation rows, two weight blocks
constexpr int kHwSfCol = kHwTileN;               // scale columns behind the accumulator, two buffers of 16
template <bool kPair> struct HwCfg {
  static constexpr int kStages = kPair ? 6 : 4;
  static constexpr int kWRows = kPair ? kHwTileN / 2 : kHwTileN;    // weight rows in a CTA's shared memory
  static constexpr int kStageBytes = kBmmABytes + kWRows * 128;
  static constexpr int kTileM = kPair ? 2 * kBmmTileM : kBmmTileM;
  static constexpr int kSmemBytes = kStages * kStageBytes + kBmmMisc + kHwSfSlots * kHwSfSlotBytes + kHwEpiBytes + 1024;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
};

template <bool kPair>
__global__ void __launch_bounds__(kHwThreads, 1)
fmoe_matmul_block128_hw_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                               const BlockMatmulParams p) {
  using Cfg = HwCfg<kPair>;
  constexpr int kHwStages = Cfg::kStages, kHwStageBytes = Cfg::kStageBytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* misc = smem + kHwStages * kHwStageBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(misc);
  uint64_t* empty_bar = full_bar + kHwStages;
  uint64_t* sf_full_bar = empty_bar + kHwStages;        // [kHwSfSlots]
  uint64_t* sf_empty_bar = sf_full_bar + kHwSfSlots;
  uint64_t* acc_full_bar = sf_empty_bar + kHwSfSlots;
  uint64_t* acc_empty_bar = acc_full_bar + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint8_t* sf_ring = misc + kBmmMisc;
  uint32_t* epi = reinterpret_cast<uint32_t*>(sf_ring + kHwSfSlots * kHwSfSlotBytes);

  const int warp = ptx::warp_index();
  const int lane = threadIdx.x & 31;
  const uint32_t rank = kPair ? ptx::cluster_ctarank() : 0u;
  const int first_tile = kPair ? blockIdx.x >> 1 : blockIdx.x, tile_step = kPair ? gridDim.x >> 1 : gridDim.x;
  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&tm_a);
    ptx::prefetch_tensormap(&tm_w);
    for (int i = 0; i < kHwStages; ++i) {
      ptx::mbar_init(ptx::smem_u32(&full_bar[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&empty_bar[i]), 1);
    }
    for (int i = 0; i < kHwSfSlots; ++i) {
      ptx::mbar_init(ptx::smem_u32(&sf_full_bar[i]), kPair ? 2 : 1);    // both CTAs' images
      ptx::mbar_init(ptx::smem_u32(&sf_empty_bar[i]), 1);
    }
    ptx::mbar_init(ptx::smem_u32(acc_full_bar), 1);
    ptx::mbar_init(ptx::smem_u32(acc_empty_bar), kPair ? 2 * kHwEpiWarps : kHwEpiWarps);
    *abort_flag = 0;
    ptx::fence_barrier_init();
    ptx::fence_proxy_async();
  }
  if (warp == 1) {
    if (kPair) {
      ptx::tmem_alloc_pair(ptx::smem_u32(tmem_slot), 512);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(ptx::smem_u32(tmem_slot), 512);
      ptx::tmem_relinquish();
    }
  }
  ptx::pdl_wait();
  ptx::tc_fence_before();
  if (kPair) ptx::cluster_sync_all();      // both CTAs' barriers are initialised before anyone signals them
  else __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int total_tiles = p.m_blocks * p.n_blocks;
  const int groups = (p.kb + 3) >> 2;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    const uint32_t full_own = ptx::smem_u32(full_bar), empty0 = ptx::smem_u32(empty_bar), smem0 = ptx::smem_u32(smem);
    const uint32_t full0 = kPair ? ptx::map_to_rank(full_own, 0) : full_own;      // both CTAs' bytes go to rank 0
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step) {
      const BlockTile at = decode_block_tile<Cfg::kTileM>(tile, p.m_blocks, p.n_blocks);
      const int m0 = at.m * Cfg::kTileM + static_cast<int>(rank) * kBmmTileM;
      const int n0 = at.n * kHwTileN + static_cast<int>(rank) * Cfg::kWRows;
      for (int k = 0; k < p.kb; ++k) {
        if (!ptx::mbar_wait(empty0 + 8 * stage, phase ^ 1u, abort_flag)) { ok = false; break; }
        if (ptx::elect_one()) {
          const uint32_t full = full0 + 8 * stage, sa = smem0 + stage * kHwStageBytes;
          if (kPair) {
            if (rank == 0) ptx::mbar_arrive_expect_tx(full_own + 8 * stage, 2 * kHwStageBytes);
            ptx::tma_load_2d_pair(sa, &tm_a, full, k * 128, m0);
            ptx::tma_load_2d_pair(sa + kBmmABytes, &tm_w, full, k * 128, n0);
          } else {
            ptx::mbar_arrive_expect_tx(full, kHwStageBytes);
            ptx::tma_load_2d(sa, &tm_a, full, k * 128, m0);
            ptx::tma_load_2d(sa + kBmmABytes, &tm_w, full, k * 128, n0);
          }
        }
        __syncwarp();
        if (++stage == kHwStages) { stage = 0; phase ^= 1u; }
      }
    }
    if (!ok && lane == 0) bmm_fail<kPair>(p.status, abort_flag, 0x21);
    ptx::pdl_release();
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------------ MMA issuer: four K blocks at a time
    const uint32_t full0 = ptx::smem_u32(full_bar), empty0 = ptx::smem_u32(empty_bar);
    const uint32_t sf_full0 = ptx::smem_u32(sf_full_bar), sf_empty0 = ptx::smem_u32(sf_empty_bar), sf0 = ptx::smem_u32(sf_ring);
    const uint32_t acc_full = ptx::smem_u32(acc_full_bar), acc_empty = ptx::smem_u32(acc_empty_bar);
    // commits of a pair arrive in both CTAs
    const uint32_t empty_peer = kPair ? ptx::map_to_rank(empty0, 1) : 0u, sf_empty_peer = kPair ? ptx::map_to_rank(sf_empty0, 1) : 0u;
    auto commit = [](uint32_t own, uint32_t peer) {
      if (kPair) {
        ptx::umma_commit_pair(own);
        ptx::umma_commit_pair(peer);
      } else {
        ptx::umma_commit(own);
      }
    };
    constexpr uint64_t kDesc = ptx::sw128_kmajor_desc_template();
    const uint64_t da0 = ptx::make_smem_desc(kDesc, ptx::smem_u32(smem));
    const uint64_t db0 = ptx::make_smem_desc(kDesc, ptx::smem_u32(smem) + kBmmABytes);
    int stage = 0, slot = 0;
    uint32_t phase = 0, slot_phase = 0, acc_phase = 0, buf = 0;
    bool ok = true;
    for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step) {
      if (!ptx::mbar_wait(acc_empty, acc_phase ^ 1u, abort_flag)) { ok = false; break; }
      acc_phase ^= 1u;
      ptx::tc_fence_after();
      for (int g = 0; ok && g < groups; ++g) {
        if (!(kPair ? ptx::mbar_wait_cluster(sf_full0 + 8 * slot, slot_phase, abort_flag)
                    : ptx::mbar_wait(sf_full0 + 8 * slot, slot_phase, abort_flag))) { ok = false; break; }
        ptx::tc_fence_after();
        const uint32_t sfa = tmem_base + kHwSfCol + buf * 16, sfb = sfa + 4;
        if (ptx::elect_one()) {
          const uint32_t src = sf0 + slot * kHwSfSlotBytes;
          if (kPair) {
            ptx::tmem_cp_32x128b_warpx4_pair(sfa, ptx::make_rows16_desc(src));
            ptx::tmem_cp_32x128b_warpx4_pair(sfb, ptx::make_rows16_desc(src + 512));
            ptx::tmem_cp_32x128b_warpx4_pair(sfb + 4, ptx::make_rows16_desc(src + 1024));
          } else {
            ptx::tmem_cp_32x128b_warpx4(sfa, ptx::make_rows16_desc(src));
            ptx::tmem_cp_32x128b_warpx4(sfb, ptx::make_rows16_desc(src + 512));
            ptx::tmem_cp_32x128b_warpx4(sfb + 4, ptx::make_rows16_desc(src + 1024));
          }
          commit(sf_empty0 + 8 * slot, sf_empty_peer + 8 * slot);        // the images may be overwritten once copied
        }
        __syncwarp();
        if (++slot == kHwSfSlots) { slot = 0; slot_phase ^= 1u; }
        buf ^= 1u;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (4 * g + u >= p.kb) break;
          if (!ptx::mbar_wait(full0 + 8 * stage, phase, abort_flag)) { ok = false; break; }
          ptx::tc_fence_after();
          if (ptx::elect_one()) {
            const uint64_t da = da0 + static_cast<uint32_t>(stage * (kHwStageBytes >> 4));
            const uint64_t db = db0 + static_cast<uint32_t>(stage * (kHwStageBytes >> 4));
            const uint32_t idesc = ptx::idesc_with_scale_byte(p.idesc, u);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              if (kPair) ptx::umma_mxf8_block_scale_pair(tmem_base, da + kk * 2, db + kk * 2, idesc, sfa, sfb, (g | u | kk) ? 1u : 0u);
              else ptx::umma_mxf8_block_scale(tmem_base, da + kk * 2, db + kk * 2, idesc, sfa, sfb, (g | u | kk) ? 1u : 0u);
            commit(empty0 + 8 * stage, empty_peer + 8 * stage);
          }
          __syncwarp();
          if (++stage == kHwStages) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) break;
      if (ptx::elect_one()) commit(acc_full, kPair ? ptx::map_to_rank(acc_full, 1) : 0u);
      __syncwarp();
    }
    if (!ok && lane == 0) bmm_fail<kPair>(p.status, abort_flag, 0x22);
  } else if (warp == 2 || warp == 3) {
    // ------------------------------------------------------------------ scale images
    // Two warps take the groups of four K blocks in turn: one alone, with a load's latency and an arrival
    // at the peer for each group, was slower than the MMAs of a pair (220 us for 8192 x 4096 x 7168 instead
    // of 209, both without bands).
    const uint32_t sf_own = ptx::smem_u32(sf_full_bar), sf_empty0 = ptx::smem_u32(sf_empty_bar);
    const uint32_t sf_full0 = kPair ? ptx::map_to_rank(sf_own, 0) : sf_own;
    const int nb = (p.n + 127) >> 7;
    const size_t pitch = static_cast<size_t>(scale_pitch(p.kb));
    static_assert(kHwSfSlots == 4, "each warp goes to and fro between two slots");
    int slot = warp - 2, g = warp - 2;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step, g -= groups) {
      const BlockTile at = decode_block_tile<Cfg::kTileM>(tile, p.m_blocks, p.n_blocks);
      const int m0 = at.m * Cfg::kTileM + static_cast<int>(rank) * kBmmTileM, nb0 = at.n * 2;
      const float* w0 = p.w_scale + static_cast<size_t>(nb0) * p.kb;
      const float* w1 = p.w_scale + static_cast<size_t>(min(nb0 + 1, nb - 1)) * p.kb;
      for (; g < groups; g += 2) {
        // loads first, so that their latency overlaps the wait for a free slot
        uint32_t a[4], w[2] = {0u, 0u};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = m0 + 32 * r + lane;
          a[r] = row < p.m ? __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(p.a_scale) + row * pitch + 4 * g)) : 0u;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (4 * g + j < p.kb) {      // a power of two's biased exponent is its byte
            w[0] |= ((__float_as_uint(__ldg(w0 + 4 * g + j)) >> 23) & 0xffu) << (8 * j);
            w[1] |= ((__float_as_uint(__ldg(w1 + 4 * g + j)) >> 23) & 0xffu) << (8 * j);
          }
        if (!ptx::mbar_wait(sf_empty0 + 8 * slot, phase ^ 1u, abort_flag)) { ok = false; break; }
        uint4* dst = reinterpret_cast<uint4*>(sf_ring + slot * kHwSfSlotBytes);
        dst[lane] = make_uint4(a[0], a[1], a[2], a[3]);
        dst[32 + lane] = make_uint4(w[0], w[0], w[0], w[0]);
        dst[64 + lane] = make_uint4(w[1], w[1], w[1], w[1]);
        ptx::fence_proxy_async();      // generic-proxy stores above are read by tcgen05.cp
        __syncwarp();
        if (kPair) {
          if (lane == 0) ptx::mbar_arrive_cluster(sf_full0 + 8 * slot);
          __syncwarp();
        } else {
          ptx::mbar_arrive_if(sf_full0 + 8 * slot, lane == 0);
        }
        if (slot >= 2) phase ^= 1u;
        slot ^= 2;
      }
    }
    if (!ok && lane == 0) bmm_fail<kPair>(p.status, abort_flag, 0x23);
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ drain and epilogue
    const uint32_t acc_full = ptx::smem_u32(acc_full_bar), acc_empty_own = ptx::smem_u32(acc_empty_bar);
    const uint32_t acc_empty = kPair ? ptx::map_to_rank(acc_empty_own, 0) : acc_empty_own;
    const int quad = warp & 3, half = (warp - 4) >> 2;
    uint32_t* mine = epi + (warp - 4) * (32 * kBmmEpiPitch);
    const uint32_t t = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(half * 128);
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = first_tile; tile < total_tiles; tile += tile_step) {
      const BlockTile at = decode_block_tile<Cfg::kTileM>(tile, p.m_blocks, p.n_blocks);
      const int m0 = at.m * Cfg::kTileM + static_cast<int>(rank) * kBmmTileM, n0 = at.n * kHwTileN;
      if (!ptx::mbar_wait(acc_full, phase, abort_flag, p.kb)) { ok = false; break; }
      phase ^= 1u;
      ptx::tc_fence_after();
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32(t + c * 32, v[c]);
      ptx::tmem_ld_wait();
      ptx::tc_fence_before();
      if (kPair) {                                       // the next tile may use the accumulator
        if (lane == 0) ptx::mbar_arrive_cluster_relaxed(acc_empty);
        __syncwarp();
      } else {
        ptx::mbar_arrive_if(acc_empty, lane == 0);
      }
      float acc[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) acc[j] = __uint_as_float(v[j >> 5][j & 31]);
      store_rows_bf16<128>(acc, mine, p.out, m0 + quad * 32, p.m, n0 + half * 128, p.n);
    }
    if (!ok && threadIdx.x == 128) bmm_fail<kPair>(p.status, abort_flag, 0x24);
  }

  ptx::tc_fence_before();
  if (kPair) ptx::cluster_sync_all();      // neither CTA leaves while its partner can still signal it or read its shared memory
  else __syncthreads();
  ptx::settle(abort_flag);
  if (warp == 1) {
    ptx::tc_fence_after();
    if (kPair) ptx::tmem_dealloc_pair(tmem_base, 512);
    else ptx::tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace fmoe
