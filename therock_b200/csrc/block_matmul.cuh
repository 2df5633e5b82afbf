// Product of e4m3 matrices with one scale per 128 of K on the activations' rows and per 128 x 128
// block on the weights:
//   out[i, j] = sum_b sa[i, b] sw[j / 128, b] P_b[i, j],   P_b = sum_{k in block b} a[i, k] w[j, k]
//
// The scales change with every block of K, so P_b is a fresh accumulator in tensor memory (one pipeline
// stage: 128 elements of K) and eight epilogue warps add it, scaled, to running sums in registers:
// acc += P_b * (sa * sw), the product of the scales rounded to 32 bits.  Warp (quadrant q, half h) owns row 32q + lane and columns 128h .. 128h + 127,
// one weight block.
//
// What bounds it is instructions and their latencies, not the MMAs (512 cycles a stage): issuing a
// stage's MMAs and commits behind two waits takes a warp 600 to 800 cycles next to busy neighbours, and
// every instruction that an epilogue warp spends besides its multiply-adds counts twice on each
// scheduler.  So four warps issue, one to each of four 128-column accumulators (half of the tile, parity
// of the stage), and the epilogue's loop takes four K blocks at a time with all addresses and parities in
// registers.
//
// Large products are also bound by power.  There two CTAs share a tile of 256 rows (kPair): each holds its
// own 128 activation rows and half of the weight rows, so that a third less comes from L2 and the MMAs
// read a third less of shared memory, and the tiles go through the result in bands.
//
// Measured on a B200, 8192 x 4096 x 7168: 201 to 205 us = 2390 TFLOP/s in a short run; back to back under the power
// limit 237 us = 2030 TFLOP/s at 1410 MHz (one CTA to a tile: 212 and 253 at 1360 MHz; without bands 219 and
// 260).  A library e4m3 product without block scales takes 195 us back to back.  In a short run and without
// bands one issuing warp and one 256-column accumulator per stage took 245 us, sixteen epilogue warps of 64
// columns 272, and 192-column tiles whose accumulator is read at once 246.
//
// A separate warp loads the scales of four blocks at a time, multiplies the activations' by those of the
// tile's two weight blocks and leaves the products in shared memory.
#pragma once

#include <cuda_bf16.h>

#include "ptx.cuh"
#include "scales.cuh"

namespace fmoe {

constexpr int kBmmThreads = 512;          // warps 0, 1: TMA, scales; 4-7: MMA; 8-15: epilogue
constexpr int kBmmEpiWarps = 8;
constexpr int kBmmTileM = 128, kBmmTileN = 256;
constexpr int kBmmABytes = kBmmTileM * 128;
constexpr int kBmmScaleSlots = 2;         // ring of scale products, four K blocks a slot
constexpr int kBmmScaleSlotFloats = 4 * 2 * kBmmTileM;
constexpr int kBmmEpiPitch = 8;           // words: 16 bf16 columns of a row
constexpr int kBmmEpiBytes = kBmmEpiWarps * 32 * kBmmEpiPitch * 4;
constexpr int kBmmMisc = 256;
template <bool kPair> struct BmmCfg {
  static constexpr int kHalfRows = kPair ? 64 : 128;        // weight rows of half a tile in a CTA's shared memory
  static constexpr int kStageBytes = kBmmABytes + 2 * kHalfRows * 128;
  static constexpr int kTileM = kPair ? 2 * kBmmTileM : kBmmTileM;
  static constexpr int kStages = 4;                         // six for a pair cost 1.3 % (8192 x 4096 x 7168)
  static constexpr int kUsedBytes = kStages * kStageBytes + kBmmMisc + kBmmScaleSlots * kBmmScaleSlotFloats * 4 + kBmmEpiBytes + 1024;
  // A CTA takes all of its SM's tensor memory, and a pair holds one SM's while it waits for the other's.
  // With this much shared memory nothing that uses tensor memory is on an SM at the same time (a cluster
  // of the kernel for few rows, on another stream, could hold the one and wait for the other).
  static constexpr int kSmemBytes = kUsedBytes < 184 * 1024 ? 184 * 1024 : kUsedBytes;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
};
// setmaxnreg redistributes the 512 x 128 registers of the launch: what the roles take must not exceed it.
constexpr int kBmmThinRegs = 80, kBmmIssueRegs = 40, kBmmFatRegs = 184;
static_assert(128 * (kBmmThinRegs + kBmmIssueRegs) + 256 * kBmmFatRegs <= kBmmThreads * 128, "register budget");

enum : int { kStatusBmmTimeout = 0x600 };

struct BlockMatmulParams {
  const void* a_scale;      // f32 [m, kb] or UE8M0 bytes [m, scale_pitch(kb)]
  const float* w_scale;     // [ceil(n / 128), kb]
  int m, n, kb;             // kb: blocks of 128 along K
  int m_blocks, n_blocks;   // tiles
  __nv_bfloat16* out;
  int* status;              // may be null
  uint32_t idesc;
};

// Tile order: bands of 1024 rows, in a band column by column.  The tiles that run side by side then read
// 1024 rows and a few thousand columns, half of what a single band of 8192 rows made them read (and 218 ->
// 210 us for 8192 x 4096 x 7168 with power-of-two scales; bands of 2048 and 4096 rows are as good).
struct BlockTile {
  int m, n;                 // in tiles
};
template <int kTileM>
__device__ __forceinline__ BlockTile decode_block_tile(int tile, int m_blocks, int n_blocks) {
  constexpr int kBand = 1024 / kTileM;
  const int band = tile / (kBand * n_blocks), local = tile - band * (kBand * n_blocks);
  const int height = min(kBand, m_blocks - band * kBand), n = local / height;
  return {band * kBand + local - n * height, n};
}

static __device__ int g_bmm_status;      // for calls without a status word

// kPair: both CTAs of a pair give up.
template <bool kPair>
__device__ __noinline__ void bmm_fail(int* status, volatile int* abort_flag, int code) {
  atomicExch(status != nullptr ? status : &g_bmm_status, kStatusBmmTimeout | code);
  if (kPair) ptx::raise_in_peer(abort_flag);
}

// Exponent byte -> power of two (0 is 2^-127, 255 is NaN).
__device__ __forceinline__ float ue8m0_value(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : (byte == 255u ? 0x7fffffffu : byte << 23));
}

// A warp's 32 rows x kCols columns (lane = row) to bf16, one rounding: 16 columns at a time turn through
// the warp's area of shared memory so that two lanes write 32 consecutive bytes of a row.
template <int kCols>
__device__ __forceinline__ void store_rows_bf16(const float (&acc)[kCols], uint32_t* area, __nv_bfloat16* out, int row0, int rows,
                                                int col0, int n) {
  const int lane = threadIdx.x & 31;
  const bool vec_out = (n & 7) == 0;
#pragma unroll
  for (int c = 0; c < kCols / 16; ++c) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(acc[c * 16 + 2 * j], acc[c * 16 + 2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&b);
    }
    __syncwarp();
    uint4* dst = reinterpret_cast<uint4*>(area + lane * kBmmEpiPitch);
    dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
    dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
    __syncwarp();
#pragma unroll
    for (int it = 0; it < 2; ++it) {
      const int r = it * 16 + (lane >> 1);
      const int col = col0 + c * 16 + (lane & 1) * 8;
      if (row0 + r < rows && col < n) {
        const uint4 val = *reinterpret_cast<const uint4*>(area + r * kBmmEpiPitch + (lane & 1) * 4);
        __nv_bfloat16* o = out + static_cast<size_t>(row0 + r) * n + col;
        if (vec_out) {
          *reinterpret_cast<uint4*>(o) = val;
        } else {
          const uint32_t x[4] = {val.x, val.y, val.z, val.w};
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (col + e < n) reinterpret_cast<uint16_t*>(o)[e] = static_cast<uint16_t>(x[e >> 1] >> (16 * (e & 1)));
        }
      }
    }
  }
}

template <bool kPair>
__global__ void __launch_bounds__(kBmmThreads, 1)
fmoe_matmul_block128_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                            const BlockMatmulParams p) {
  using Cfg = BmmCfg<kPair>;
  constexpr int kBmmStages = Cfg::kStages, kBmmStageBytes = Cfg::kStageBytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* misc = smem + kBmmStages * kBmmStageBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(misc);
  uint64_t* empty_bar = full_bar + kBmmStages;
  uint64_t* part_full_bar = empty_bar + kBmmStages;      // [half][parity]
  uint64_t* part_empty_bar = part_full_bar + 4;          // [half][parity]
  uint64_t* sc_full_bar = part_empty_bar + 4;            // [kBmmScaleSlots]
  uint64_t* sc_empty_bar = sc_full_bar + kBmmScaleSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sc_empty_bar + kBmmScaleSlots);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* sc_ring = reinterpret_cast<float*>(misc + kBmmMisc);
  uint32_t* epi = reinterpret_cast<uint32_t*>(sc_ring + kBmmScaleSlots * kBmmScaleSlotFloats);

  const int warp = ptx::warp_index();
  const int lane = threadIdx.x & 31;
  const uint32_t rank = kPair ? ptx::cluster_ctarank() : 0u;
  const int first_tile = kPair ? blockIdx.x >> 1 : blockIdx.x, tile_step = kPair ? gridDim.x >> 1 : gridDim.x;
  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&tm_a);
    ptx::prefetch_tensormap(&tm_w);
    for (int i = 0; i < kBmmStages; ++i) {
      ptx::mbar_init(ptx::smem_u32(&full_bar[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&empty_bar[i]), 2);      // both halves' MMAs
    }
    for (int b = 0; b < 4; ++b) {
      ptx::mbar_init(ptx::smem_u32(&part_full_bar[b]), 1);
      ptx::mbar_init(ptx::smem_u32(&part_empty_bar[b]), kPair ? kBmmEpiWarps : kBmmEpiWarps / 2);
    }
    for (int i = 0; i < kBmmScaleSlots; ++i) {
      ptx::mbar_init(ptx::smem_u32(&sc_full_bar[i]), 32);
      ptx::mbar_init(ptx::smem_u32(&sc_empty_bar[i]), kBmmEpiWarps);
    }
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

  if (warp < 4) {
    ptx::setmaxnreg_dec<kBmmThinRegs>();
    if (warp == 0) {
      // ---------------------------------------------------------------- TMA producer
      const uint32_t full_own = ptx::smem_u32(full_bar), empty0 = ptx::smem_u32(empty_bar), smem0 = ptx::smem_u32(smem);
      const uint32_t full0 = kPair ? ptx::map_to_rank(full_own, 0) : full_own;      // both CTAs' bytes go to rank 0
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step) {
        const BlockTile at = decode_block_tile<Cfg::kTileM>(tile, p.m_blocks, p.n_blocks);
        const int m0 = at.m * Cfg::kTileM + static_cast<int>(rank) * kBmmTileM;
        const int n0 = at.n * kBmmTileN + static_cast<int>(rank) * Cfg::kHalfRows;
        for (int k = 0; k < p.kb; ++k) {
          if (!ptx::mbar_wait(empty0 + 8 * stage, phase ^ 1u, abort_flag)) { ok = false; break; }
          if (ptx::elect_one()) {
            const uint32_t full = full0 + 8 * stage, sa = smem0 + stage * kBmmStageBytes;
            if (kPair) {
              if (rank == 0) ptx::mbar_arrive_expect_tx(full_own + 8 * stage, 2 * kBmmStageBytes);
              ptx::tma_load_2d_pair(sa, &tm_a, full, k * 128, m0);
              ptx::tma_load_2d_pair(sa + kBmmABytes, &tm_w, full, k * 128, n0);
              ptx::tma_load_2d_pair(sa + kBmmABytes + Cfg::kHalfRows * 128, &tm_w, full, k * 128, n0 + 128);
            } else {
              ptx::mbar_arrive_expect_tx(full, kBmmStageBytes);
              ptx::tma_load_2d(sa, &tm_a, full, k * 128, m0);
              ptx::tma_load_2d(sa + kBmmABytes, &tm_w, full, k * 128, n0);
            }
          }
          __syncwarp();
          if (++stage == kBmmStages) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok && lane == 0) bmm_fail<kPair>(p.status, abort_flag, 0x01);
      ptx::pdl_release();
    } else if (warp == 1) {
      // ---------------------------------------------------------------- scale products
      int slot = 0;
      uint32_t sphase = 0;
      bool ok = true;
      const int nb = (p.n + 127) >> 7;
      const bool vec = (p.kb & 3) == 0 && (reinterpret_cast<uintptr_t>(p.a_scale) & 15) == 0;
      for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step) {
        const BlockTile at = decode_block_tile<Cfg::kTileM>(tile, p.m_blocks, p.n_blocks);
        const int m0 = at.m * Cfg::kTileM + static_cast<int>(rank) * kBmmTileM, nb0 = at.n * 2;
        const float* sw0 = p.w_scale + static_cast<size_t>(nb0) * p.kb;
        const float* sw1 = p.w_scale + static_cast<size_t>(min(nb0 + 1, nb - 1)) * p.kb;
        for (int k = 0; k < p.kb; k += 4) {
          float w0[4], w1[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            w0[j] = k + j < p.kb ? __ldg(sw0 + k + j) : 0.0f;
            w1[j] = k + j < p.kb ? __ldg(sw1 + k + j) : 0.0f;
          }
          float s[4][4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = m0 + 32 * r + lane;
#pragma unroll
            for (int j = 0; j < 4; ++j) s[r][j] = 0.0f;
            if (row < p.m) {
              const float* src = static_cast<const float*>(p.a_scale) + static_cast<size_t>(row) * p.kb + k;
              if (vec) {
                const float4 v = __ldg(reinterpret_cast<const float4*>(src));
                s[r][0] = v.x; s[r][1] = v.y; s[r][2] = v.z; s[r][3] = v.w;
              } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  if (k + j < p.kb) s[r][j] = __ldg(src + j);
              }
            }
          }
          if (!ptx::mbar_wait(ptx::smem_u32(&sc_empty_bar[slot]), sphase ^ 1u, abort_flag)) { ok = false; break; }
          float* dst = sc_ring + slot * kBmmScaleSlotFloats;
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              dst[(2 * j) * kBmmTileM + 32 * r + lane] = s[r][j] * w0[j];
              dst[(2 * j + 1) * kBmmTileM + 32 * r + lane] = s[r][j] * w1[j];
            }
          ptx::mbar_arrive(ptx::smem_u32(&sc_full_bar[slot]));
          if (++slot == kBmmScaleSlots) { slot = 0; sphase ^= 1u; }
        }
      }
      if (!ok && lane == 0) bmm_fail<kPair>(p.status, abort_flag, 0x03);
    }
  } else if (warp < 8) {
    ptx::setmaxnreg_dec<kBmmIssueRegs>();
    // ------------------------------------------------------------------ MMA issuers
    const int half = (warp >> 1) & 1, parity = warp & 1;
    static_assert(kBmmStages % 2 == 0, "an issuer has the stages of its parity");
    const uint32_t full0 = ptx::smem_u32(full_bar) + 8 * parity, empty0 = ptx::smem_u32(empty_bar) + 8 * parity;
    const uint32_t part_full = ptx::smem_u32(part_full_bar) + 8 * (2 * half + parity), part_empty = ptx::smem_u32(part_empty_bar) + 8 * (2 * half + parity);
    constexpr uint64_t kDesc = ptx::sw128_kmajor_desc_template();
    const uint32_t smem0 = ptx::smem_u32(smem) + parity * kBmmStageBytes;
    const uint64_t da0 = ptx::make_smem_desc(kDesc, smem0);
    const uint64_t db0 = ptx::make_smem_desc(kDesc, smem0 + kBmmABytes + half * Cfg::kHalfRows * 128);
    const uint32_t d_tmem = tmem_base + half * 256 + parity * 128;
    const int my_tiles = rank == 0 && first_tile < total_tiles ? (total_tiles - 1 - first_tile) / tile_step + 1 : 0;
    const uint32_t part_full_peer = kPair ? ptx::map_to_rank(part_full, 1) : 0u, empty_peer = kPair ? ptx::map_to_rank(empty0, 1) : 0u;
    const long long stages = static_cast<long long>(my_tiles) * p.kb;
    uint32_t phase = 0, part_phase = 1;
    bool ok = true;
    for (long long it = parity; ok && it < stages; it += kBmmStages) {
#pragma unroll
      for (int h = 0; h < kBmmStages / 2; ++h) {             // stages parity, parity + 2, ...
        if (it + 2 * h >= stages) break;
        if (!ptx::mbar_wait(full0 + 16 * h, phase, abort_flag) || !ptx::mbar_wait(part_empty, part_phase, abort_flag)) { ok = false; break; }
        part_phase ^= 1u;
        ptx::tc_fence_after();
        if (ptx::elect_one()) {
          constexpr uint32_t kTwo = (2 * kBmmStageBytes) >> 4;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            if (kPair) ptx::umma_f8_pair(d_tmem, da0 + (h * kTwo + kk * 2), db0 + (h * kTwo + kk * 2), p.idesc, kk ? 1u : 0u);
            else ptx::umma_f8(d_tmem, da0 + (h * kTwo + kk * 2), db0 + (h * kTwo + kk * 2), p.idesc, kk ? 1u : 0u);
          }
          if (kPair) {      // in both CTAs
            ptx::umma_commit_pair(part_full);
            ptx::umma_commit_pair(part_full_peer);
            ptx::umma_commit_pair(empty0 + 16 * h);
            ptx::umma_commit_pair(empty_peer + 16 * h);
          } else {
            ptx::umma_commit(part_full);
            ptx::umma_commit(empty0 + 16 * h);
          }
        }
        __syncwarp();
      }
      phase ^= 1u;
    }
    if (!ok && lane == 0) bmm_fail<kPair>(p.status, abort_flag, 0x02);
  } else {
    // ------------------------------------------------------------------ promotion and epilogue
    ptx::setmaxnreg_inc<kBmmFatRegs>();
    const int quad = warp & 3;
    const int half = (warp - 8) >> 2;
    uint32_t* mine = epi + (warp - 8) * (32 * kBmmEpiPitch);
    // x is the accumulator that the first and the third of four K blocks are in, y the other one.
    const uint32_t part_full0 = ptx::smem_u32(part_full_bar) + 16 * half, part_empty_own = ptx::smem_u32(part_empty_bar) + 16 * half;
    const uint32_t part_empty0 = kPair ? ptx::map_to_rank(part_empty_own, 0) : part_empty_own;      // the issuers are in rank 0
    uint32_t full_x = part_full0, full_y = part_full0 + 8, empty_x = part_empty0, empty_y = part_empty0 + 8;
    uint32_t t_x = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(half * 256), t_y = t_x + 128;
    uint32_t phase_x = 0, phase_y = 0;
    static_assert(kBmmScaleSlots == 2, "the scale slots alternate");
    uint32_t sc_full_now = ptx::smem_u32(sc_full_bar), sc_full_next = sc_full_now + 8;
    uint32_t sc_empty_now = ptx::smem_u32(sc_empty_bar), sc_empty_next = sc_empty_now + 8;
    int slot_now = 0, slot_next = kBmmScaleSlotFloats;
    uint32_t sc_phase = 0;                               // of both slots: flips every two groups
    const int kb = p.kb, m_blocks = p.m_blocks, n_blocks = p.n_blocks;
    const bool leader = lane == 0;
    const float* sc_base = sc_ring + half * kBmmTileM + quad * 32 + lane;
    bool ok = true;
    for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step) {
      const BlockTile at = decode_block_tile<Cfg::kTileM>(tile, m_blocks, n_blocks);
      const int m0 = at.m * Cfg::kTileM + static_cast<int>(rank) * kBmmTileM, n0 = at.n * kBmmTileN;
      float acc[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) acc[j] = 0.0f;
#pragma unroll 1
      for (int k0 = 0; k0 < kb; k0 += 4) {
        if (!ptx::mbar_wait(sc_full_now, sc_phase, abort_flag)) { ok = false; break; }
        float sc[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) sc[u] = sc_base[slot_now + 2 * u * kBmmTileM];
        __syncwarp();
        ptx::mbar_arrive_if(sc_empty_now, leader);
        if (slot_now != 0) sc_phase ^= 1u;
        const uint32_t f = sc_full_now, e = sc_empty_now;
        const int sl = slot_now;
        sc_full_now = sc_full_next; sc_full_next = f;
        sc_empty_now = sc_empty_next; sc_empty_next = e;
        slot_now = slot_next; slot_next = sl;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (k0 + u < kb) {
            if (!ptx::mbar_wait((u & 1) ? full_y : full_x, (u & 1) ? phase_y : phase_x, abort_flag)) { ok = false; break; }
            ptx::tc_fence_after();
            const uint32_t t = (u & 1) ? t_y : t_x;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t v[32];
              ptx::tmem_ld_32x32(t + c * 32, v);
              ptx::tmem_ld_wait();
              if (c == 3) {      // everything has left this accumulator: the MMAs may overwrite it
                ptx::tc_fence_before();
                if (kPair) ptx::mbar_arrive_cluster_relaxed_if((u & 1) ? empty_y : empty_x, leader);
                else ptx::mbar_arrive_if((u & 1) ? empty_y : empty_x, leader);
                if (u & 1) phase_y ^= 1u; else phase_x ^= 1u;
              }
#pragma unroll
              for (int j = 0; j < 32; ++j) acc[c * 32 + j] = fmaf(__uint_as_float(v[j]), sc[u], acc[c * 32 + j]);
            }
          }
        }
        if (!ok) break;
      }
      if (kb & 1) {      // the next tile starts with the other accumulator
        uint32_t x;
        x = full_x; full_x = full_y; full_y = x;
        x = empty_x; empty_x = empty_y; empty_y = x;
        x = t_x; t_x = t_y; t_y = x;
        x = phase_x; phase_x = phase_y; phase_y = x;
      }
      if (!ok) break;
      store_rows_bf16<128>(acc, mine, p.out, m0 + quad * 32, p.m, n0 + half * 128, p.n);
    }
    if (!ok && threadIdx.x == 256) bmm_fail<kPair>(p.status, abort_flag, 0x04);
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
