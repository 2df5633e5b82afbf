// The e4m3 product with power-of-two block scales (see block_matmul.cuh for the arithmetic): the tensor
// core applies the scales itself (tcgen05.mma kind::mxf8f6f4.block_scale), so one 128 x 256 accumulator
// stays in tensor memory for the whole K loop and nothing is promoted in registers.
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
// Measured on a B200, 8192 x 4096 x 7168: 181 to 187 us = 2570 to 2660 TFLOP/s, what a library e4m3 product
// without block scales sustains (2606) under the power limit that bounds both; the promotion in
// registers takes 219 us.
#pragma once

#include "block_matmul.cuh"

namespace fmoe {

constexpr int kHwThreads = 384;                   // warps 0-3: TMA, MMA, scale images, idle; warps 4-11: epilogue
constexpr int kHwEpiWarps = 8;
constexpr int kHwTileN = 256;
constexpr int kHwStages = 4;
constexpr int kHwStageBytes = kBmmABytes + kHwTileN * 128;
constexpr int kHwEpiBytes = kHwEpiWarps * 32 * kBmmEpiPitch * 4;
constexpr int kHwSfSlots = 4;                     // ring of scale images, four K blocks a slot
constexpr int kHwSfSlotBytes = 512 + 2 * 512;     // activation rows, two weight blocks
constexpr int kHwSfCol = kHwTileN;               // scale columns behind the accumulator, two buffers of 16
constexpr int kHwSmemBytes = kHwStages * kHwStageBytes + kBmmMisc + kHwSfSlots * kHwSfSlotBytes + kHwEpiBytes + 1024;
static_assert(kHwSmemBytes <= 227 * 1024, "shared memory budget");

__global__ void __launch_bounds__(kHwThreads, 1)
fmoe_matmul_block128_hw_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                               const BlockMatmulParams p) {
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
  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&tm_a);
    ptx::prefetch_tensormap(&tm_w);
    for (int i = 0; i < kHwStages; ++i) {
      ptx::mbar_init(ptx::smem_u32(&full_bar[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&empty_bar[i]), 1);
    }
    for (int i = 0; i < kHwSfSlots; ++i) {
      ptx::mbar_init(ptx::smem_u32(&sf_full_bar[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&sf_empty_bar[i]), 1);
    }
    ptx::mbar_init(ptx::smem_u32(acc_full_bar), 1);
    ptx::mbar_init(ptx::smem_u32(acc_empty_bar), kHwEpiWarps);
    *abort_flag = 0;
    ptx::fence_barrier_init();
    ptx::fence_proxy_async();
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_slot), 512);
    ptx::tmem_relinquish();
  }
  ptx::pdl_wait();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int total_tiles = p.m_blocks * p.n_blocks;
  const int groups = (p.kb + 3) >> 2;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    const uint32_t full0 = ptx::smem_u32(full_bar), empty0 = ptx::smem_u32(empty_bar), smem0 = ptx::smem_u32(smem);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < total_tiles; tile += gridDim.x) {
      const int m0 = tile % p.m_blocks * kBmmTileM, n0 = tile / p.m_blocks * kHwTileN;
      for (int k = 0; k < p.kb; ++k) {
        if (!ptx::mbar_wait(empty0 + 8 * stage, phase ^ 1u, abort_flag)) { ok = false; break; }
        if (ptx::elect_one()) {
          const uint32_t full = full0 + 8 * stage, sa = smem0 + stage * kHwStageBytes;
          ptx::mbar_arrive_expect_tx(full, kHwStageBytes);
          ptx::tma_load_2d(sa, &tm_a, full, k * 128, m0);
          ptx::tma_load_2d(sa + kBmmABytes, &tm_w, full, k * 128, n0);
        }
        __syncwarp();
        if (++stage == kHwStages) { stage = 0; phase ^= 1u; }
      }
    }
    if (!ok && lane == 0) bmm_fail(p.status, 0x21);
    ptx::pdl_release();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer: four K blocks at a time
    static_assert(kHwStages == 4, "a group of four K blocks goes once round the stages");
    const uint32_t full0 = ptx::smem_u32(full_bar), empty0 = ptx::smem_u32(empty_bar);
    const uint32_t sf_full0 = ptx::smem_u32(sf_full_bar), sf_empty0 = ptx::smem_u32(sf_empty_bar), sf0 = ptx::smem_u32(sf_ring);
    const uint32_t acc_full = ptx::smem_u32(acc_full_bar), acc_empty = ptx::smem_u32(acc_empty_bar);
    constexpr uint64_t kDesc = ptx::sw128_kmajor_desc_template();
    const uint64_t da0 = ptx::make_smem_desc(kDesc, ptx::smem_u32(smem));
    const uint64_t db0 = ptx::make_smem_desc(kDesc, ptx::smem_u32(smem) + kBmmABytes);
    int stage = 0, slot = 0;
    uint32_t phase = 0, slot_phase = 0, acc_phase = 0, buf = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < total_tiles; tile += gridDim.x) {
      if (!ptx::mbar_wait(acc_empty, acc_phase ^ 1u, abort_flag)) { ok = false; break; }
      acc_phase ^= 1u;
      ptx::tc_fence_after();
      for (int g = 0; ok && g < groups; ++g) {
        if (!ptx::mbar_wait(sf_full0 + 8 * slot, slot_phase, abort_flag)) { ok = false; break; }
        ptx::tc_fence_after();
        const uint32_t sfa = tmem_base + kHwSfCol + buf * 16, sfb = sfa + 4;
        if (ptx::elect_one()) {
          const uint32_t src = sf0 + slot * kHwSfSlotBytes;
          ptx::tmem_cp_32x128b_warpx4(sfa, ptx::make_rows16_desc(src));
          ptx::tmem_cp_32x128b_warpx4(sfb, ptx::make_rows16_desc(src + 512));
          ptx::tmem_cp_32x128b_warpx4(sfb + 4, ptx::make_rows16_desc(src + 1024));
          ptx::umma_commit(sf_empty0 + 8 * slot);        // the image may be overwritten once copied
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
              ptx::umma_mxf8_block_scale(tmem_base, da + kk * 2, db + kk * 2, idesc, sfa, sfb, (g | u | kk) ? 1u : 0u);
            ptx::umma_commit(empty0 + 8 * stage);
          }
          __syncwarp();
          if (++stage == kHwStages) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) break;
      if (ptx::elect_one()) ptx::umma_commit(acc_full);
      __syncwarp();
    }
    if (!ok && lane == 0) bmm_fail(p.status, 0x22);
  } else if (warp == 2) {
    // ------------------------------------------------------------------ scale images
    const uint32_t sf_full0 = ptx::smem_u32(sf_full_bar), sf_empty0 = ptx::smem_u32(sf_empty_bar);
    const int nb = (p.n + 127) >> 7;
    const size_t pitch = static_cast<size_t>(scale_pitch(p.kb));
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < total_tiles; tile += gridDim.x) {
      const int m0 = tile % p.m_blocks * kBmmTileM, nb0 = tile / p.m_blocks * 2;
      const float* w0 = p.w_scale + static_cast<size_t>(nb0) * p.kb;
      const float* w1 = p.w_scale + static_cast<size_t>(min(nb0 + 1, nb - 1)) * p.kb;
      for (int g = 0; g < groups; ++g) {
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
        ptx::mbar_arrive_if(sf_full0 + 8 * slot, lane == 0);
        if (++slot == kHwSfSlots) { slot = 0; phase ^= 1u; }
      }
    }
    if (!ok && lane == 0) bmm_fail(p.status, 0x23);
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ drain and epilogue
    const uint32_t acc_full = ptx::smem_u32(acc_full_bar), acc_empty = ptx::smem_u32(acc_empty_bar);
    const int quad = warp & 3, half = (warp - 4) >> 2;
    uint32_t* mine = epi + (warp - 4) * (32 * kBmmEpiPitch);
    const uint32_t t = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(half * 128);
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x) {
      const int m0 = tile % p.m_blocks * kBmmTileM, n0 = tile / p.m_blocks * kHwTileN;
      if (!ptx::mbar_wait(acc_full, phase, abort_flag)) { ok = false; break; }
      phase ^= 1u;
      ptx::tc_fence_after();
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32(t + c * 32, v[c]);
      ptx::tmem_ld_wait();
      ptx::tc_fence_before();
      ptx::mbar_arrive_if(acc_empty, lane == 0);         // the next tile may use the accumulator
      float acc[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) acc[j] = __uint_as_float(v[j >> 5][j & 31]);
      store_rows_bf16<128>(acc, mine, p.out, m0 + quad * 32, p.m, n0 + half * 128, p.n);
    }
    if (!ok && threadIdx.x == 128) bmm_fail(p.status, 0x24);
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace fmoe
