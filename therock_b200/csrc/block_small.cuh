// The e4m3 product with block scales for few activation rows (see block_matmul.cuh for the arithmetic).
//
// With few rows the weights are the work: they are read once and every byte is used for a handful of
// multiply-adds.  So the weights are the MMA's M side -- 128 weight rows, exactly one block of their
// scales -- and the activation rows its N side, kNT = 16, 32 or 128 of them, which keeps the
// activations' share of the traffic small.  Lane = output column, accumulator column = row.  P_b of a
// block of K is a kNT-column accumulator, several of which are in flight, and the epilogue warps add
// them, scaled, in registers: a row's scale times the weight block's comes from shared memory, the
// same for all lanes.
//
// Where the tiles alone do not fill the GPU, the K blocks of a tile are shared out over a cluster of
// 2, 4 or 8 CTAs.  Each adds up its blocks, sends every CTA its share of the columns through
// distributed shared memory, and sums the shares it received in the order of the ranks: one launch, no
// workspace, the same bits every time.
//
// Measured on a B200: 16 x 18432 x 7168 in 23.5 us = 5650 GB/s (memory-bound: 88 % of a copy's rate, the
// rest is launch and the first block's way), 1 x 4096 x 2048 in 3.6 us, 16 x 4096 x 7168 in 7.0 (four CTAs to
// a tile), 64 x 7744 x 2048 in 7.6.  The kernels with 128 x 256 tiles take 36 to 40 us for the first of these
// shapes, 22 to 26 for the third and 8.5 to 10 for the last.
#pragma once

#include <cuda_bf16.h>

#include "block_matmul.cuh"

namespace fmoe {

constexpr int kBsWBytes = 128 * 128;
constexpr int kBsScaleSlots = 4;              // ring of scale products, four K blocks a slot
constexpr int kBsMaxStages = 10;
constexpr int kBsMisc = 512;
constexpr int kBsMostSmem = 220 * 1024;

template <int kNT> struct BlockSmallCfg {
  static constexpr int kGroups = kNT > 64 ? 2 : 1;            // groups of four epilogue warps
  static constexpr int kCols = kNT / kGroups;                 // accumulator columns of a thread
  static constexpr int kThreads = 128 + 128 * kGroups;
  static constexpr int kBufs = kNT <= 32 ? 8 : 4;             // accumulators in flight
  static constexpr int kTmemCols = kNT * kBufs;               // 128, 256 or 512
  // No two CTAs may wait for each other's tensor memory while they hold their own (a CTA of a cluster
  // waits for its peers): with at least this much shared memory to a CTA, those that fit an SM together
  // never ask for more than its 512 columns.
  static constexpr int kMinSmem = (kTmemCols == 128 ? 56 : kTmemCols == 256 ? 113 : 200) * 1024;
  static constexpr int kStageBytes = kBsWBytes + kNT * 128;
  static constexpr int kScaleBytes = kBsScaleSlots * 4 * kNT * 4;
  static_assert(184 * 1024 + kMinSmem > 227 * 1024, "not beside a CTA of a pair (see BmmCfg)");
  static_assert(kTmemCols == 128 || kTmemCols == 256 || kTmemCols == 512, "see kMinSmem");
  static constexpr int smem_bytes(int stages, bool split) {
    return stages * kStageBytes + kBsMisc + kScaleBytes + (split ? kNT * 128 * 4 : 0) + 1024;
  }
};

struct BlockSmallParams {
  const void* a_scale;      // f32 [m, kb] or UE8M0 bytes [m, scale_pitch(kb)]
  const float* w_scale;     // [ceil(n / 128), kb]
  int m, n, kb;
  int t_tiles;              // tiles of kNT activation rows
  int split;                // CTAs (one cluster) that share a tile's K blocks
  int stages;
  __nv_bfloat16* out;
  int* status;              // may be null
  uint32_t idesc;
};

template <int kNT, bool kBytes>
__global__ void __launch_bounds__(BlockSmallCfg<kNT>::kThreads)
fmoe_matmul_block128_small_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                                  const BlockSmallParams p) {
  using Cfg = BlockSmallCfg<kNT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* misc = smem + p.stages * Cfg::kStageBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(misc);            // [kBsMaxStages]
  uint64_t* empty_bar = full_bar + kBsMaxStages;                     // [kBsMaxStages]
  uint64_t* part_full_bar = empty_bar + kBsMaxStages;                // [kBufs]
  uint64_t* part_empty_bar = part_full_bar + 8;                      // [kBufs]
  uint64_t* sc_full_bar = part_empty_bar + 8;                        // [kBsScaleSlots]
  uint64_t* sc_empty_bar = sc_full_bar + kBsScaleSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sc_empty_bar + kBsScaleSlots);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* sc_ring = reinterpret_cast<float*>(misc + kBsMisc);
  float* red = sc_ring + Cfg::kScaleBytes / 4;                       // [split][kNT / split][128]

  const int warp = ptx::warp_index();
  const int lane = threadIdx.x & 31;
  const int rank = p.split > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  const int tile = blockIdx.x / p.split;
  const int t0 = tile % p.t_tiles * kNT, n_blk = tile / p.t_tiles;
  const int k0 = static_cast<int>(static_cast<long long>(p.kb) * rank / p.split);
  const int k1 = static_cast<int>(static_cast<long long>(p.kb) * (rank + 1) / p.split);

  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&tm_a);
    ptx::prefetch_tensormap(&tm_w);
    for (int i = 0; i < p.stages; ++i) {
      ptx::mbar_init(ptx::smem_u32(&full_bar[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&empty_bar[i]), 1);
    }
    for (int i = 0; i < Cfg::kBufs; ++i) {
      ptx::mbar_init(ptx::smem_u32(&part_full_bar[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&part_empty_bar[i]), 4 * Cfg::kGroups);
    }
    for (int i = 0; i < kBsScaleSlots; ++i) {
      ptx::mbar_init(ptx::smem_u32(&sc_full_bar[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&sc_empty_bar[i]), 4 * Cfg::kGroups);
    }
    *abort_flag = 0;
    ptx::fence_barrier_init();
    ptx::fence_proxy_async();
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_slot), Cfg::kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::pdl_wait();
  ptx::tc_fence_before();
  if (p.split > 1) ptx::cluster_sync_all();      // every CTA of the cluster runs before any writes to its shared memory
  else __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    const uint32_t full0 = ptx::smem_u32(full_bar), empty0 = ptx::smem_u32(empty_bar), smem0 = ptx::smem_u32(smem);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int k = k0; k < k1; ++k) {
      if (!ptx::mbar_wait(empty0 + 8 * stage, phase ^ 1u, abort_flag)) { ok = false; break; }
      if (ptx::elect_one()) {
        const uint32_t full = full0 + 8 * stage, sw = smem0 + stage * Cfg::kStageBytes;
        ptx::mbar_arrive_expect_tx(full, Cfg::kStageBytes);
        ptx::tma_load_2d(sw, &tm_w, full, k * 128, n_blk * 128);
        ptx::tma_load_2d(sw + kBsWBytes, &tm_a, full, k * 128, t0);
      }
      __syncwarp();
      if (++stage == p.stages) { stage = 0; phase ^= 1u; }
    }
    if (!ok && lane == 0) bmm_fail<false>(p.status, abort_flag, 0x11);
    ptx::pdl_release();
  } else if (warp & 1 && warp < 4) {
    // ------------------------------------------------------------------ MMA issuers
    // Two warps take turns, as a stage's waits, MMAs and commits keep one for longer than its MMAs take:
    // this one has the blocks of one parity, and the accumulators of that parity.
    const int mine = warp >> 1;
    const uint32_t full0 = ptx::smem_u32(full_bar), empty0 = ptx::smem_u32(empty_bar);
    const uint32_t part_full0 = ptx::smem_u32(part_full_bar), part_empty0 = ptx::smem_u32(part_empty_bar);
    constexpr uint64_t kDesc = ptx::sw128_kmajor_desc_template();
    const uint64_t da0 = ptx::make_smem_desc(kDesc, ptx::smem_u32(smem));
    const uint64_t db0 = ptx::make_smem_desc(kDesc, ptx::smem_u32(smem) + kBsWBytes);
    const int stages = p.stages;
    int stage = mine;
    uint32_t phase = 0, buf_phase = 1;
    if (stage >= stages) { stage -= stages; phase = 1; }
    bool ok = true;
    for (int k = k0 + mine; ok && k < k1; k += Cfg::kBufs) {
#pragma unroll
      for (int h = 0; h < Cfg::kBufs; h += 2) {
        if (k + h >= k1) break;
        if (!ptx::mbar_wait(full0 + 8 * stage, phase, abort_flag) ||
            !ptx::mbar_wait(part_empty0 + 8 * (mine + h), buf_phase, abort_flag)) { ok = false; break; }
        ptx::tc_fence_after();
        if (ptx::elect_one()) {
          const uint64_t da = da0 + static_cast<uint32_t>(stage * (Cfg::kStageBytes >> 4));
          const uint64_t db = db0 + static_cast<uint32_t>(stage * (Cfg::kStageBytes >> 4));
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) ptx::umma_f8(tmem_base + (mine + h) * kNT, da + kk * 2, db + kk * 2, p.idesc, kk ? 1u : 0u);
          ptx::umma_commit(part_full0 + 8 * (mine + h));
          ptx::umma_commit(empty0 + 8 * stage);
        }
        __syncwarp();
        stage += 2;
        while (stage >= stages) { stage -= stages; phase ^= 1u; }
      }
      buf_phase ^= 1u;
    }
    if (!ok && lane == 0) bmm_fail<false>(p.status, abort_flag, 0x12);
  } else if (warp == 2) {
    // ------------------------------------------------------------------ scale products
    // The next slot is requested before the present one is handed over: two slots, eight blocks of K, are
    // on their way from the start.
    constexpr int kR = (kNT + 31) / 32;
    const uint32_t sc_full0 = ptx::smem_u32(sc_full_bar), sc_empty0 = ptx::smem_u32(sc_empty_bar);
    const float* sw = p.w_scale + static_cast<size_t>(n_blk) * p.kb;
    const int pitch = scale_pitch(p.kb);
    const bool vec = !kBytes && (p.kb & 3) == 0 && (k0 & 3) == 0 && ((k1 - k0) & 3) == 0 && (reinterpret_cast<uintptr_t>(p.a_scale) & 15) == 0;
    float s[2][kR][4], w[2][4];
    auto request = [&](int k, float (&sv)[kR][4], float (&wv)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        wv[j] = k + j < k1 ? __ldg(sw + k + j) : 0.0f;
        // power-of-two scales go by their exponent alone, as in the kernel whose MMAs apply them
        if (kBytes) wv[j] = ue8m0_value((__float_as_uint(wv[j]) >> 23) & 0xffu);
      }
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        const int t = t0 + 32 * r + lane;
        const bool live = t < p.m && 32 * r + lane < kNT;
        if (kBytes) {
          // four bytes from any position: two aligned words of the row (its pitch is a multiple of four)
          uint32_t lo = 0u, hi = 0u;
          if (live && k < k1) {
            const uint32_t* words = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(p.a_scale) + static_cast<size_t>(t) * pitch);
            lo = __ldg(words + (k >> 2));
            if ((k & 3) != 0 && (k >> 2) + 1 < (pitch >> 2)) hi = __ldg(words + (k >> 2) + 1);
          }
          const uint32_t four = __funnelshift_r(lo, hi, 8 * (k & 3));
#pragma unroll
          for (int j = 0; j < 4; ++j) sv[r][j] = live && k + j < k1 ? ue8m0_value((four >> (8 * j)) & 0xffu) : 0.0f;
        } else if (vec) {
          float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
          if (live && k < k1) f = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.a_scale) + static_cast<size_t>(t) * p.kb + k));
          sv[r][0] = f.x; sv[r][1] = f.y; sv[r][2] = f.z; sv[r][3] = f.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            sv[r][j] = live && k + j < k1 ? __ldg(static_cast<const float*>(p.a_scale) + static_cast<size_t>(t) * p.kb + k + j) : 0.0f;
        }
      }
    };
    bool ok = true;
    int n = 0;                              // slots handed over
    auto hand_over = [&](int k, float (&sv)[kR][4], float (&wv)[4]) {
      const int slot = n % kBsScaleSlots;
      if (!ptx::mbar_wait(sc_empty0 + 8 * slot, ((n / kBsScaleSlots) & 1u) ^ 1u, abort_flag)) { ok = false; return; }
      float* dst = sc_ring + slot * 4 * kNT;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < kR; ++r)
          if (32 * r + lane < kNT) dst[j * kNT + 32 * r + lane] = sv[r][j] * wv[j];
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(sc_full0 + 8 * slot);
      __syncwarp();
      ++n;
    };
    int k = k0;
    request(k, s[0], w[0]);
    for (; ok && k < k1; k += 8) {
      request(k + 4, s[1], w[1]);
      hand_over(k, s[0], w[0]);
      if (!ok || k + 4 >= k1) break;
      request(k + 8, s[0], w[0]);
      hand_over(k + 4, s[1], w[1]);
    }
    if (!ok && lane == 0) bmm_fail<false>(p.status, abort_flag, 0x13);
  }

  float acc[Cfg::kCols];
  const int quad = warp & 3;
  const int col0 = warp >= 4 ? ((warp - 4) >> 2) * Cfg::kCols : 0;
  const int row = quad * 32 + lane;                                  // output column within the tile
  if (warp >= 4) {
    // ------------------------------------------------------------------ promotion
    const uint32_t part_full0 = ptx::smem_u32(part_full_bar), part_empty0 = ptx::smem_u32(part_empty_bar);
    const uint32_t sc_full0 = ptx::smem_u32(sc_full_bar), sc_empty0 = ptx::smem_u32(sc_empty_bar);
    const uint32_t t_base = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(col0);
    const float* sc_base = sc_ring + col0;
    int group = 0;
    bool ok = true;
#pragma unroll
    for (int j = 0; j < Cfg::kCols; ++j) acc[j] = 0.0f;
    // four K blocks at a time: a slot of scales, and accumulators whose addresses do not change
#pragma unroll 1
    for (int k = k0; k < k1; k += 4, ++group) {
      const int slot = group % kBsScaleSlots, buf0 = (group * 4) % Cfg::kBufs;
      const uint32_t phase = (group * 4 / Cfg::kBufs) & 1u;
      if (!ptx::mbar_wait(sc_full0 + 8 * slot, (group / kBsScaleSlots) & 1u, abort_flag)) { ok = false; break; }
      const float4* sc = reinterpret_cast<const float4*>(sc_base + slot * 4 * kNT);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (k + u < k1) {
          if (!ptx::mbar_wait(part_full0 + 8 * (buf0 + u), phase, abort_flag)) { ok = false; break; }
          ptx::tc_fence_after();
          // the whole accumulator is read before anything is added, so it is free again at once
          uint32_t v[Cfg::kCols];
          const uint32_t t = t_base + (buf0 + u) * kNT;
          if constexpr (Cfg::kCols == 16) {
            ptx::tmem_ld_32x16(t, reinterpret_cast<uint32_t(&)[16]>(v[0]));
          } else {
#pragma unroll
            for (int c = 0; c < Cfg::kCols; c += 32) ptx::tmem_ld_32x32(t + c, reinterpret_cast<uint32_t(&)[32]>(v[c]));
          }
          ptx::tmem_ld_wait();
          ptx::tc_fence_before();
          ptx::mbar_arrive_if(part_empty0 + 8 * (buf0 + u), lane == 0);
#pragma unroll
          for (int q = 0; q < Cfg::kCols / 4; ++q) {
            const float4 f = sc[u * (kNT / 4) + q];
            acc[4 * q] = fmaf(__uint_as_float(v[4 * q]), f.x, acc[4 * q]);
            acc[4 * q + 1] = fmaf(__uint_as_float(v[4 * q + 1]), f.y, acc[4 * q + 1]);
            acc[4 * q + 2] = fmaf(__uint_as_float(v[4 * q + 2]), f.z, acc[4 * q + 2]);
            acc[4 * q + 3] = fmaf(__uint_as_float(v[4 * q + 3]), f.w, acc[4 * q + 3]);
          }
        }
      }
      if (!ok) break;
      __syncwarp();
      ptx::mbar_arrive_if(sc_empty0 + 8 * slot, lane == 0);
    }
    if (!ok && threadIdx.x == 128) bmm_fail<false>(p.status, abort_flag, 0x14);
  }

  const int out_col = n_blk * 128 + row;
  if (p.split == 1) {
    if (warp >= 4 && out_col < p.n) {
#pragma unroll
      for (int j = 0; j < Cfg::kCols; ++j)
        if (t0 + col0 + j < p.m) p.out[static_cast<size_t>(t0 + col0 + j) * p.n + out_col] = __float2bfloat16_rn(acc[j]);
    }
  } else {
    // ------------------------------------------------------------------ sum over the cluster
    // Rank r sums the columns c with c % split == r, so that a tile with few live rows keeps every CTA
    // busy; the sums of four columns are in flight at a time.
    const int log_split = 31 - __clz(p.split), share = kNT >> log_split;
    if (warp >= 4) {
      const uint32_t red0 = ptx::smem_u32(red) + static_cast<uint32_t>((rank * share) * 128 + row) * 4u;
#pragma unroll
      for (int j = 0; j < Cfg::kCols; ++j) {
        const int c = col0 + j;
        if (t0 + c >= p.m) break;
        const uint32_t dst = ptx::map_to_rank(red0 + static_cast<uint32_t>((c >> log_split) * 512), static_cast<uint32_t>(c & (p.split - 1)));
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(acc[j]) : "memory");
      }
    }
    ptx::cluster_sync_all();
    if (warp >= 4) {
      const int first = ((warp - 4) >> 2) * (share / Cfg::kGroups);
      for (int j0 = first; j0 < first + share / Cfg::kGroups; j0 += 4) {
        if (t0 + (j0 << log_split) + rank >= p.m) break;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        for (int r = 0; r < p.split; ++r) {
          const float* src = red + (r * share + j0) * 128 + row;
#pragma unroll
          for (int j = 0; j < 4; ++j) sum[j] += j0 + j < share ? src[j * 128] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int t = t0 + ((j0 + j) << log_split) + rank;
          if (j0 + j < first + share / Cfg::kGroups && t < p.m && out_col < p.n)
            p.out[static_cast<size_t>(t) * p.n + out_col] = __float2bfloat16_rn(sum[j]);
        }
      }
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  ptx::settle(abort_flag);
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

}  // namespace fmoe
