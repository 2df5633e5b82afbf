// Products grouped by expert for sm_100a, ragged in the rows, as operators with gradients.
//
//   rows kernel   out[r, :] = W_g x[r, :]   (kWMnMajor = false: W [G, N, K], contraction over K)
//                 out[r, :] = W_g^T x[r, :] (kWMnMajor = true: contraction over N; W is read as it
//                                            lies, the MMA takes it MN-major)
//   wgrad kernel  dW_g = sum_r dy[r, :]^T x[r, :], both operands MN-major, contraction over the
//                 group's rows
//
// Both are persistent kernels of CTA pairs (cta_group::2, 256 x 256 tiles, 64 elements of the
// contraction per stage, six stages in the rows kernel and five in the wgrad kernel, two 256-column
// accumulators in tensor memory), with the roles of the pair kernel of the fused operator: producer
// warp, MMA warp, four epilogue warps.  A tile's contraction is one pair's, whatever its length.
//
// Rows kernel: the weights are the MMA's M side and the rows its N side.  M tiles of weights are
// always full, and N goes in steps of 32, so a group of any size costs its own rows rounded up to
// 32 instead of to 256.  A group of s rows is cut into ceil(s / 256) chunks of equal size.
// Rows of a neighbouring group that come along in the last 32 only produce accumulator columns
// that nobody stores.
//
// Measured on a B200 (bf16; 1644 TFLOP/s and 6457 GB/s are what a library product and a copy reach there):
//   8192 rows in 8 equal groups x 28672 x 4096: 1.21 to 1.33 ms = 1450 to 1586 TFLOP/s in a short run, 1.36 to
//   1.50 under the power limit; 8192 rows in 32 equal groups x 4096 x 7168: y and dx 0.37 to 0.40 ms, 1200 to
//   1290 TFLOP/s with the weights coming from memory at 5 TB/s (their loads alone take 0.31 ms, the MMAs
//   alone 0.23), 0.49 under the power limit; dw 0.48 ms = 1010 TFLOP/s (loads, MMAs and the 1.9 GB of stores
//   take 0.34 to 0.39 ms in any two of the three), 0.56 under the power limit; 31 groups of uneven sizes
//   take 0.46, 0.46 and 0.56 ms, and 0.57, 0.56 and 0.64 under the power limit; 32 rows over 8 groups x 28672 x
//   4096: 0.295 ms = 6370 GB/s; 2 rows through 1024 x 512: 4.85 us.
// What it took: roles that run as whole warps with one elected thread (a lane-0 branch made the issue of
// the MMAs and the loads the bound: 1.75 -> 1.31 ms), a store phase without a branch per store (-> 1.21), and
// no cluster-scope release in a loop (dw 0.76 -> 0.49).  Prefetching the weights into L2 seven to sixteen
// stages ahead made y 3 to 9 % slower.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace fmoe {

constexpr int kGrpThreads = 192;
constexpr int kGrpMaxGroups = 1024;
constexpr int kGrpStages = 6;
constexpr int kGrpOperandBytes = 128 * 128;                 // 128 rows (or two 64-column chunks x 64 rows) x 128 bytes
constexpr int kGrpStageBytes = 2 * kGrpOperandBytes;
constexpr int kGrpStageK = 64;                              // 16-bit elements of the contraction per stage
constexpr int kGrpTile = 256;
constexpr int kGrpMisc = 256 + 2 * (kGrpMaxGroups + 8) * 4; // barriers, group starts, cumulative chunks
constexpr int kGrpSmemBytes = kGrpStages * kGrpStageBytes + kGrpMisc + 1024;
// wgrad: one stage less, which leaves room for two 64-column x 32-row store buffers per epilogue warp
constexpr int kWgThreads = kGrpThreads + 32;                // and a warp for ragged last stages
constexpr int kWgStages = 5;
constexpr int kWgStoreBytes = 32 * 128;
constexpr int kWgSmemBytes = kWgStages * kGrpStageBytes + 4 * 2 * kWgStoreBytes + kGrpMisc + 1024;
static_assert(kGrpSmemBytes <= 227 * 1024 && kWgSmemBytes <= 227 * 1024, "shared memory budget");

enum : int { kStatusGroupedTimeout = 0x500 };

struct GroupedParams {
  const int32_t* offsets;   // [groups + 1]
  int groups;
  int rows;
  int m_blocks;             // rows kernel: 256-wide blocks of output columns; wgrad: blocks of N
  int k_blocks;             // wgrad: 256-wide blocks of K
  int k_iters;              // rows kernel: stages per tile
  int n, k;                 // wgrad: dimensions of dw; rows kernel: n = output columns
  uint16_t* out;
  int* status;              // may be null
  uint32_t idesc;           // instruction descriptor without N (rows kernel) / complete (wgrad)
};

template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if (kBf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

static __device__ int g_grouped_status;      // for calls without a status word

static __device__ __noinline__ void grouped_fail(int* status, volatile int* abort_flag, int code) {
  atomicExch(status != nullptr ? status : &g_grouped_status, kStatusGroupedTimeout | code);
  ptx::raise_in_peer(abort_flag);
}

// One warp: starts[0 .. G] = running maximum of the offsets clamped to [0, rows];
// cum[0 .. G] = cumulative number of `chunk`-row pieces.
__device__ __forceinline__ void scan_groups(const int32_t* offsets, int groups, int rows, int chunk, int* starts, int* cum) {
  const int lane = threadIdx.x & 31;
  int run_start = min(max(offsets[0], 0), rows), run_cum = 0;
  if (lane == 0) { starts[0] = run_start; cum[0] = 0; }
  for (int g0 = 0; g0 < groups; g0 += 32) {
    const int g = g0 + lane;
    int end = g < groups ? min(max(offsets[g + 1], 0), rows) : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, end, d);
      if (lane >= d) end = max(end, o);
    }
    end = max(end, run_start);
    int start = __shfl_up_sync(0xffffffffu, end, 1);
    if (lane == 0) start = run_start;
    int c = g < groups ? (end - start + chunk - 1) / chunk : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, c, d);
      if (lane >= d) c += o;
    }
    c += run_cum;
    if (g < groups) { starts[g + 1] = end; cum[g + 1] = c; }
    run_start = __shfl_sync(0xffffffffu, end, 31);
    run_cum = __shfl_sync(0xffffffffu, c, 31);
  }
}

struct RowsTile {
  int group, m_blk;
  int row0, live;           // first row of the chunk, rows of it
  int n;                    // MMA columns: live rounded up to 32
};

// Tile order: group, then block of output columns, then the group's chunks: CTA pairs that run
// side by side read the same weights, once from memory and then from L2.
__device__ __forceinline__ RowsTile decode_rows_tile(int tile, const int* starts, const int* cum, int groups, int m_blocks) {
  int lo = 1, hi = groups;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (static_cast<long long>(cum[mid]) * m_blocks > tile) hi = mid; else lo = mid + 1;
  }
  RowsTile t;
  t.group = lo - 1;
  const int cnt = cum[lo] - cum[lo - 1];
  const int local = tile - cum[lo - 1] * m_blocks;
  t.m_blk = local / cnt;
  const int chunk = local % cnt;
  const int size = starts[lo] - starts[lo - 1];
  // equal chunks in steps of 32; the last one is never empty (fewer than 32 * cnt rows are lost to
  // the rounding, and only where cnt < 8, since the chunks are 256 long otherwise)
  const int per = ((size + cnt - 1) / cnt + 31) & ~31;
  t.row0 = starts[lo - 1] + chunk * per;
  t.live = min(per, size - chunk * per);
  t.n = (t.live + 31) & ~31;
  return t;
}

template <int kStages, int kStoreBytes>
struct GroupedSmem {
  uint8_t *stages, *store;
  uint64_t *full_bar, *empty_bar, *acc_full_bar, *acc_empty_bar, *tail_bar, *peer_bar;
  uint32_t* tmem_slot;
  volatile int* abort_flag;
  int *starts, *cum;

  __device__ __forceinline__ explicit GroupedSmem(uint8_t* raw) {
    stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    store = stages + kStages * kGrpStageBytes;
    uint8_t* misc = store + kStoreBytes;
    full_bar = reinterpret_cast<uint64_t*>(misc);       // used in rank 0
    empty_bar = full_bar + kStages;                     // both ranks
    acc_full_bar = empty_bar + kStages;                 // [2] both ranks
    acc_empty_bar = acc_full_bar + 2;                   // [2] used in rank 0
    tail_bar = acc_empty_bar + 2;                       // [kStages] wgrad: this CTA's bytes of a ragged stage
    peer_bar = tail_bar + kStages;                      // [kStages] used in rank 0: the peer's ragged stage is ready
    tmem_slot = reinterpret_cast<uint32_t*>(peer_bar + kStages);
    abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    starts = reinterpret_cast<int*>(misc + 256);
    cum = starts + kGrpMaxGroups + 8;
  }

  // Barriers, tensor memory, group table.
  __device__ __forceinline__ uint32_t setup(const GroupedParams& p, int warp) const {
    if (threadIdx.x == 0) {
      for (int i = 0; i < kStages; ++i) {
        ptx::mbar_init(ptx::smem_u32(&full_bar[i]), 1);
        ptx::mbar_init(ptx::smem_u32(&empty_bar[i]), 1);
        ptx::mbar_init(ptx::smem_u32(&tail_bar[i]), 1);
        ptx::mbar_init(ptx::smem_u32(&peer_bar[i]), 1);
      }
      for (int b = 0; b < 2; ++b) {
        ptx::mbar_init(ptx::smem_u32(&acc_full_bar[b]), 1);
        ptx::mbar_init(ptx::smem_u32(&acc_empty_bar[b]), 8);      // 4 epilogue warps in each CTA
      }
      *abort_flag = 0;
      ptx::fence_barrier_init();
      ptx::fence_proxy_async();
    }
    if (warp == 1) {
      ptx::tmem_alloc_pair(ptx::smem_u32(tmem_slot), 512);
      ptx::tmem_relinquish_pair();
    }
    ptx::pdl_wait();              // the offsets and operands of this call are read from here on
    if (warp == 2) scan_groups(p.offsets, p.groups, p.rows, kGrpTile, starts, cum);
    ptx::tc_fence_before();
    ptx::cluster_sync_all();      // both CTAs' barriers are initialised before anyone signals them
    ptx::tc_fence_after();
    return *tmem_slot;
  }
};

__device__ __forceinline__ void grouped_teardown(uint32_t tmem_base, int warp, const volatile int* abort_flag) {
  // neither CTA leaves while its partner can still signal its barriers or read its shared memory
  ptx::tc_fence_before();
  ptx::cluster_sync_all();
  ptx::settle(abort_flag);
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem_base, 512);
  }
}

// Tensor maps of the row matrix with boxes of 128, 64, 32 and 16 rows: a chunk's half, a multiple
// of 16 up to 128, is the sum of at most four of them.
struct RowMaps {
  CUtensorMap m[4];
};

template <bool kBf16, bool kWMnMajor>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGrpThreads, 1)
fmoe_grouped_rows_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ RowMaps tm_x,
                         const GroupedParams p) {
  extern __shared__ uint8_t smem_raw[];
  const GroupedSmem<kGrpStages, 0> s(smem_raw);
  const int warp = ptx::warp_index();
  const int lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();
  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&tm_w);
    for (int i = 0; i < 4; ++i) ptx::prefetch_tensormap(&tm_x.m[i]);
  }
  const uint32_t tmem_base = s.setup(p, warp);
  const int total_tiles = s.cum[p.groups] * p.m_blocks;
  const int first_tile = blockIdx.x >> 1;
  const int tile_step = gridDim.x >> 1;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (both ranks)
    const uint32_t full0 = ptx::map_to_rank(ptx::smem_u32(s.full_bar), 0);   // completion bytes of both CTAs go to rank 0
    const uint32_t full_own = ptx::smem_u32(s.full_bar), empty_own = ptx::smem_u32(s.empty_bar);
    const uint32_t smem0 = ptx::smem_u32(s.stages);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step) {
      const RowsTile t = decode_rows_tile(tile, s.starts, s.cum, p.groups, p.m_blocks);
      const int group = ptx::uniform(t.group);
      const int m0 = ptx::uniform(t.m_blk) * kGrpTile + static_cast<int>(rank) * 128;
      const int half = ptx::uniform(t.n) >> 1;
      const int r0 = ptx::uniform(t.row0) + static_cast<int>(rank) * half;
      const uint32_t bytes = 2u * (kGrpOperandBytes + half * 128);
      for (int k = 0; k < p.k_iters; ++k) {
        if (!ptx::mbar_wait(empty_own + 8 * stage, phase ^ 1u, s.abort_flag)) { ok = false; break; }
        if (ptx::elect_one()) {
          const uint32_t full = full0 + 8 * stage;
          const uint32_t sa = smem0 + stage * kGrpStageBytes;
          const int kx = k * kGrpStageK;
          if (rank == 0) ptx::mbar_arrive_expect_tx(full_own + 8 * stage, bytes);
          if (kWMnMajor) {
            ptx::tma_load_3d_pair(sa, &tm_w, full, m0, kx, group);
            ptx::tma_load_3d_pair(sa + kGrpOperandBytes / 2, &tm_w, full, m0 + 64, kx, group);
          } else {
            ptx::tma_load_3d_pair(sa, &tm_w, full, kx, m0, group);
          }
          int done = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int box = 128 >> i;
            if (half & box) {
              ptx::tma_load_2d_pair(sa + kGrpOperandBytes + done * 128, &tm_x.m[i], full, kx, r0 + done);
              done += box;
            }
          }
        }
        __syncwarp();
        if (++stage == kGrpStages) { stage = 0; phase ^= 1u; }
      }
    }
    if (!ok && lane == 0) grouped_fail(p.status, s.abort_flag, 0x01);
    ptx::pdl_release();   // all operands requested: the next kernel may begin its set-up
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (rank 0 only)
    if (rank == 0) {
      constexpr uint64_t kDescA = kWMnMajor ? ptx::sw128_mnmajor_desc_template(kGrpOperandBytes / 2)
                                            : ptx::sw128_kmajor_desc_template();
      constexpr uint64_t kDescB = ptx::sw128_kmajor_desc_template();
      // 16 elements of the contraction: 32 bytes along a swizzled row, or 16 rows of 128 bytes
      constexpr uint64_t kAdvA = kWMnMajor ? (16 * 128) >> 4 : 32 >> 4;
      const uint32_t smem0 = ptx::smem_u32(s.stages);
      const uint64_t da0 = ptx::make_smem_desc(kDescA, smem0);
      const uint64_t db0 = ptx::make_smem_desc(kDescB, smem0 + kGrpOperandBytes);
      const uint32_t full_own = ptx::smem_u32(s.full_bar), empty_own = ptx::smem_u32(s.empty_bar);
      const uint32_t empty_peer = ptx::map_to_rank(empty_own, 1);
      const uint32_t acc_full = ptx::smem_u32(s.acc_full_bar), acc_full_peer = ptx::map_to_rank(acc_full, 1);
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step) {
        const RowsTile t = decode_rows_tile(tile, s.starts, s.cum, p.groups, p.m_blocks);
        const uint32_t idesc = p.idesc | (static_cast<uint32_t>(ptx::uniform(t.n) >> 3) << 17);
        if (!ptx::mbar_wait(ptx::smem_u32(&s.acc_empty_bar[acc]), acc_phase ^ 1u, s.abort_flag)) { ok = false; break; }
        ptx::tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kGrpTile);
        for (int k = 0; k < p.k_iters; ++k) {
          if (!ptx::mbar_wait(full_own + 8 * stage, phase, s.abort_flag)) { ok = false; break; }
          ptx::tc_fence_after();
          if (ptx::elect_one()) {
            const uint64_t da = da0 + static_cast<uint32_t>(stage * (kGrpStageBytes >> 4));
            const uint64_t db = db0 + static_cast<uint32_t>(stage * (kGrpStageBytes >> 4));
#pragma unroll
            for (int kk = 0; kk < kGrpStageK / 16; ++kk)
              ptx::umma_f16_pair(d_tmem, da + kk * kAdvA, db + kk * 2, idesc, (k | kk) ? 1u : 0u);
            ptx::umma_commit_pair(empty_own + 8 * stage);
            ptx::umma_commit_pair(empty_peer + 8 * stage);
          }
          __syncwarp();
          if (++stage == kGrpStages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        if (ptx::elect_one()) {
          ptx::umma_commit_pair(acc_full + 8 * acc);
          ptx::umma_commit_pair(acc_full_peer + 8 * acc);
        }
        __syncwarp();
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
      }
      if (!ok && lane == 0) grouped_fail(p.status, s.abort_flag, 0x02);
    }
  } else {
    // ------------------------------------------------------------------ epilogue warps (both ranks)
    // Lane = output column, accumulator column = row of the result: two lanes swap halves of a
    // packed pair so that every lane stores two neighbouring columns of one row.
    const int quad = warp & 3;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step) {
      const RowsTile t = decode_rows_tile(tile, s.starts, s.cum, p.groups, p.m_blocks);
      if (!ptx::mbar_wait(ptx::smem_u32(&s.acc_full_bar[acc]), acc_phase, s.abort_flag, p.k_iters)) { ok = false; break; }
      ptx::tc_fence_after();
      const int col = t.m_blk * kGrpTile + static_cast<int>(rank) * 128 + quad * 32 + (lane & ~1);
      const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(acc * kGrpTile);
      uint16_t* o = p.out + static_cast<size_t>(t.row0 + (lane & 1)) * p.n + col;
      const size_t step = 2 * static_cast<size_t>(p.n);
      uint32_t v[2][32];
      ptx::tmem_ld_32x32(t_addr, v[0]);
      auto block = [&](uint32_t (&cur)[32], uint32_t (&next)[32], int c) {
        ptx::tmem_ld_wait();
        if (c + 32 < t.live) ptx::tmem_ld_32x32(t_addr + c + 32, next);
        uint32_t word[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const uint32_t mine = pack16<kBf16>(__uint_as_float(cur[2 * j]), __uint_as_float(cur[2 * j + 1]));
          const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, 1);
          // even lane: row 2j, columns (lane, lane + 1); odd lane: row 2j + 1, columns (lane - 1, lane)
          word[j] = (lane & 1) ? __byte_perm(other, mine, 0x7632) : __byte_perm(mine, other, 0x5410);
        }
        // one branch for the whole block: a branch per store left the shuffles unoverlapped (a
        // 256-column tile took 8.3 us, as long as 20 stages of MMAs)
        if (col < p.n) {
          if (c + 32 <= t.live) {
#pragma unroll
            for (int j = 0; j < 16; ++j) *reinterpret_cast<uint32_t*>(o + j * step) = word[j];
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (c + 2 * j + (lane & 1) < t.live) *reinterpret_cast<uint32_t*>(o + j * step) = word[j];
          }
        }
        __syncwarp();
        o += 16 * step;
      };
      for (int c = 0; c < t.live; c += 64) {
        block(v[0], v[1], c);
        if (c + 32 < t.live) block(v[1], v[0], c + 32);
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster_relaxed(ptx::map_to_rank(ptx::smem_u32(&s.acc_empty_bar[acc]), 0));
      if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
    }
    if (!ok && threadIdx.x == 64) grouped_fail(p.status, s.abort_flag, 0x03);
    // rows of no group: in front of the first one and behind the last
    const int head = s.starts[0], tail = s.starts[p.groups];
    const int vecs = p.n >> 3;
    const long long total = static_cast<long long>(head + p.rows - tail) * vecs;
    for (long long i = static_cast<long long>(blockIdx.x) * 128 + (threadIdx.x - 64); i < total; i += static_cast<long long>(gridDim.x) * 128) {
      long long r = i / vecs;
      const int v = static_cast<int>(i - r * vecs);
      if (r >= head) r += tail - head;
      *reinterpret_cast<uint4*>(p.out + static_cast<size_t>(r) * p.n + v * 8) = make_uint4(0, 0, 0, 0);
    }
  }
  grouped_teardown(tmem_base, warp, s.abort_flag);
}

// dW_g [N, K] in 256 x 256 tiles.  The contraction runs over the group's rows, 64 per stage and 16
// per MMA, from the group's first row on (a TMA box may start at any row).  The last stage issues
// only the MMAs it has rows for; where the last 16 are not full, the rest of them holds rows of the
// next group (or whatever lies behind the last one, which may be infinite or NaN), so a warp of
// each CTA overwrites those rows with zeros before the MMA may read them.  With one tile per 256
// rows of a group the result is most of the traffic: it leaves through shared memory by TMA, which
// cuts what lies outside of [N, K].
template <bool kBf16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kWgThreads, 1)
fmoe_grouped_wgrad_kernel(const __grid_constant__ CUtensorMap tm_dy, const __grid_constant__ CUtensorMap tm_x,
                          const __grid_constant__ CUtensorMap tm_dw, const GroupedParams p) {
  extern __shared__ uint8_t smem_raw[];
  const GroupedSmem<kWgStages, 4 * 2 * kWgStoreBytes> s(smem_raw);
  const int warp = ptx::warp_index();
  const int lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();
  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&tm_dy);
    ptx::prefetch_tensormap(&tm_x);
    ptx::prefetch_tensormap(&tm_dw);
  }
  const uint32_t tmem_base = s.setup(p, warp);
  const int per_group = p.m_blocks * p.k_blocks;
  const int total_tiles = p.groups * per_group;
  const int first_tile = blockIdx.x >> 1;
  const int tile_step = gridDim.x >> 1;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (both ranks)
    const uint32_t full0 = ptx::map_to_rank(ptx::smem_u32(s.full_bar), 0);
    const uint32_t full_own = ptx::smem_u32(s.full_bar), empty_own = ptx::smem_u32(s.empty_bar);
    const uint32_t tail_own = ptx::smem_u32(s.tail_bar), tail_cluster = ptx::map_to_rank(tail_own, rank);
    const uint32_t smem0 = ptx::smem_u32(s.stages);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step) {
      const int g = tile / per_group;
      const int local = tile - g * per_group;
      const int n0 = local / p.k_blocks * kGrpTile + static_cast<int>(rank) * 128;
      const int k0 = local % p.k_blocks * kGrpTile + static_cast<int>(rank) * 128;
      const int row0 = ptx::uniform(s.starts[g]);
      const int size = ptx::uniform(s.starts[g + 1]) - row0;
      for (int done = 0; done < size; done += kGrpStageK) {
        if (!ptx::mbar_wait(empty_own + 8 * stage, phase ^ 1u, s.abort_flag)) { ok = false; break; }
        const int live = min(kGrpStageK, size - done);
        const bool ragged = (live & 15) != 0;
        if (ptx::elect_one()) {
          uint32_t bar = full0 + 8 * stage;
          const uint32_t sa = smem0 + stage * kGrpStageBytes;
          if (ragged) {
            // this CTA's bytes are waited for by its tail warp
            bar = tail_cluster + 8 * stage;
            ptx::mbar_arrive_expect_tx(tail_own + 8 * stage, kGrpStageBytes);
          } else if (rank == 0) {
            ptx::mbar_arrive_expect_tx(full_own + 8 * stage, 2 * kGrpStageBytes);
          }
          const int r = row0 + done;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            ptx::tma_load_2d_pair(sa + c * (kGrpOperandBytes / 2), &tm_dy, bar, n0 + 64 * c, r);
            ptx::tma_load_2d_pair(sa + kGrpOperandBytes + c * (kGrpOperandBytes / 2), &tm_x, bar, k0 + 64 * c, r);
          }
        }
        __syncwarp();
        if (++stage == kWgStages) { stage = 0; phase ^= 1u; }
      }
    }
    if (!ok && lane == 0) grouped_fail(p.status, s.abort_flag, 0x11);
    ptx::pdl_release();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (rank 0 only)
    if (rank == 0) {
      constexpr uint64_t kDesc = ptx::sw128_mnmajor_desc_template(kGrpOperandBytes / 2);
      const uint32_t smem0 = ptx::smem_u32(s.stages);
      const uint64_t da0 = ptx::make_smem_desc(kDesc, smem0);
      const uint64_t db0 = ptx::make_smem_desc(kDesc, smem0 + kGrpOperandBytes);
      const uint32_t full_own = ptx::smem_u32(s.full_bar), empty_own = ptx::smem_u32(s.empty_bar);
      const uint32_t empty_peer = ptx::map_to_rank(empty_own, 1);
      const uint32_t acc_full = ptx::smem_u32(s.acc_full_bar), acc_full_peer = ptx::map_to_rank(acc_full, 1);
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step) {
        const int g = tile / per_group;
        const int size = ptx::uniform(s.starts[g + 1] - s.starts[g]);
        if (size == 0) continue;
        if (!ptx::mbar_wait(ptx::smem_u32(&s.acc_empty_bar[acc]), acc_phase ^ 1u, s.abort_flag)) { ok = false; break; }
        ptx::tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kGrpTile);
        for (int done = 0; done < size; done += kGrpStageK) {
          if (!ptx::mbar_wait(full_own + 8 * stage, phase, s.abort_flag)) { ok = false; break; }
          ptx::tc_fence_after();
          if (ptx::elect_one()) {
            const uint64_t da = da0 + static_cast<uint32_t>(stage * (kGrpStageBytes >> 4));
            const uint64_t db = db0 + static_cast<uint32_t>(stage * (kGrpStageBytes >> 4));
            const int live = size - done;
#pragma unroll
            for (int kk = 0; kk < kGrpStageK / 16; ++kk)
              if (kk * 16 < live) ptx::umma_f16_pair(d_tmem, da + kk * 128, db + kk * 128, p.idesc, (done | kk) ? 1u : 0u);
            ptx::umma_commit_pair(empty_own + 8 * stage);
            ptx::umma_commit_pair(empty_peer + 8 * stage);
          }
          __syncwarp();
          if (++stage == kWgStages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        if (ptx::elect_one()) {
          ptx::umma_commit_pair(acc_full + 8 * acc);
          ptx::umma_commit_pair(acc_full_peer + 8 * acc);
        }
        __syncwarp();
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
      }
      if (!ok && lane == 0) grouped_fail(p.status, s.abort_flag, 0x12);
    }
  } else if (warp == 6) {
    // ------------------------------------------------------------------ ragged last stages (both ranks)
    const uint32_t peer0 = ptx::map_to_rank(ptx::smem_u32(s.peer_bar), 0);
    int stage = 0;
    uint32_t phases = 0;            // bit i: parity of tail_bar[i] and peer_bar[i]
    bool ok = true;
    for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step) {
      const int g = tile / per_group;
      const int size = s.starts[g + 1] - s.starts[g];
      if (size == 0) continue;
      const int n_stages = (size + kGrpStageK - 1) / kGrpStageK;
      const int last_stage = (stage + n_stages - 1) % kWgStages;
      stage = (stage + n_stages) % kWgStages;
      const int live = size - (n_stages - 1) * kGrpStageK;
      if ((live & 15) == 0) continue;
      if (!ptx::mbar_wait(ptx::smem_u32(&s.tail_bar[last_stage]), (phases >> last_stage) & 1u, s.abort_flag, n_stages)) { ok = false; break; }
      const int end = (live + 15) & ~15;
      uint8_t* st = s.stages + last_stage * kGrpStageBytes;
      // four 64-column chunks (two of dy, two of x) of 64 rows x 128 bytes
      for (int i = lane; i < (end - live) * 32; i += 32) {
        const int row = live + (i >> 5);
        const int c = (i >> 3) & 3;
        *reinterpret_cast<uint4*>(st + c * (kGrpOperandBytes / 2) + row * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
      }
      ptx::fence_proxy_async();
      __syncwarp();
      // rank 1 tells rank 0, which completes the stage for the MMAs when both halves are ready
      if (rank == 1) {
        if (lane == 0) ptx::mbar_arrive_cluster(peer0 + 8 * last_stage);
      } else {
        if (!ptx::mbar_wait_cluster(ptx::smem_u32(&s.peer_bar[last_stage]), (phases >> last_stage) & 1u, s.abort_flag)) { ok = false; break; }
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&s.full_bar[last_stage]));
      }
      __syncwarp();
      phases ^= 1u << last_stage;
    }
    if (!ok && lane == 0) grouped_fail(p.status, s.abort_flag, 0x14);
  } else {
    // ------------------------------------------------------------------ epilogue warps (both ranks)
    // Lane = row n of the tile.  64 columns at a time are rounded, written to the warp's buffer in the
    // 128-byte swizzle (conflict-free) and stored as a box of 64 columns x 32 rows.
    const int quad = warp & 3;
    uint8_t* buf = s.store + quad * (2 * kWgStoreBytes);
    uint8_t* row_at = buf + lane * 128;
    const uint32_t sw = static_cast<uint32_t>(lane & 7);
    int acc = 0;
    uint32_t acc_phase = 0;
    int b = 0;
    bool ok = true;
    for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step) {
      const int g = tile / per_group;
      const int local = tile - g * per_group;
      const int n0 = local / p.k_blocks * kGrpTile + static_cast<int>(rank) * 128 + quad * 32;
      const int k0 = local % p.k_blocks * kGrpTile;
      const int size = s.starts[g + 1] - s.starts[g];
      const bool empty = size == 0;
      if (!empty) {
        if (!ptx::mbar_wait(ptx::smem_u32(&s.acc_full_bar[acc]), acc_phase, s.abort_flag, size / kGrpStageK + 1)) { ok = false; break; }
        ptx::tc_fence_after();
      }
      const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(acc * kGrpTile);
      const int cols = n0 < p.n ? min(kGrpTile, p.k - k0) : 0;
      for (int c = 0; c < cols; c += 64) {
        uint32_t v[2][32];
        if (!empty) {
          ptx::tmem_ld_32x32(t_addr + c, v[0]);
          ptx::tmem_ld_32x32(t_addr + c + 32, v[1]);
          ptx::tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[0][j] = v[1][j] = 0u;
        }
        if (lane == 0) ptx::bulk_wait_read<1>();        // the store before last has left this buffer
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const uint32_t* f = v[q >> 2] + 8 * (q & 3);
          *reinterpret_cast<uint4*>(row_at + b * kWgStoreBytes + ((static_cast<uint32_t>(q) ^ sw) << 4)) =
              make_uint4(pack16<kBf16>(__uint_as_float(f[0]), __uint_as_float(f[1])),
                         pack16<kBf16>(__uint_as_float(f[2]), __uint_as_float(f[3])),
                         pack16<kBf16>(__uint_as_float(f[4]), __uint_as_float(f[5])),
                         pack16<kBf16>(__uint_as_float(f[6]), __uint_as_float(f[7])));
        }
        ptx::fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          ptx::tma_store_3d(&tm_dw, ptx::smem_u32(buf + b * kWgStoreBytes), k0 + c, n0, g);
          ptx::bulk_commit();
        }
        __syncwarp();
        b ^= 1;
      }
      if (empty) continue;
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster_relaxed(ptx::map_to_rank(ptx::smem_u32(&s.acc_empty_bar[acc]), 0));
      if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
    }
    if (!ok && threadIdx.x == 64) grouped_fail(p.status, s.abort_flag, 0x13);
    if (lane == 0) ptx::bulk_wait<0>();
    __syncwarp();
  }
  grouped_teardown(tmem_base, warp, s.abort_flag);
}

}  // namespace fmoe
