// Host side of the e4m3 product with block scales: checks, tensor maps, launch.
#include <atomic>
#include <mutex>

#include "block_hw.cuh"
#include "block_small.cuh"

#include "host.cuh"
#include "internal.h"

namespace fmoe {
namespace {

constexpr int kMaxDevices = 64;
static_assert(kHwTileN == kBmmTileN, "one size of tile to report");

CUresult byte_map(CUtensorMap* tm, const void* base, int64_t rows, int cols, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(cols)};
  const uint32_t box[2] = {128, static_cast<uint32_t>(box_rows)};
  return encode_tensor_map(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box);
}

template <typename Kernel>
cudaError_t launch_tiles(Kernel kernel, std::atomic<bool> (&configured)[kMaxDevices], int threads, int smem, int cluster, const CUtensorMap& a,
                         const CUtensorMap& w, const BlockMatmulParams& p, int grid, cudaStream_t stream) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices || !configured[dev].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < kMaxDevices) configured[dev].store(true, std::memory_order_release);
  }
  return launch_pdl_cluster(kernel, dim3(grid), dim3(threads), smem, cluster, stream, a, w, p);
}
template <bool kPair>
cudaError_t launch_f32(const CUtensorMap& a, const CUtensorMap& w, const BlockMatmulParams& p, int grid, cudaStream_t stream) {
  static std::atomic<bool> configured[kMaxDevices] = {};
  return launch_tiles(fmoe_matmul_block128_kernel<kPair>, configured, kBmmThreads, BmmCfg<kPair>::kSmemBytes, kPair ? 2 : 1, a, w, p,
                      grid, stream);
}
template <bool kPair>
cudaError_t launch_hw(const CUtensorMap& a, const CUtensorMap& w, const BlockMatmulParams& p, int grid, cudaStream_t stream) {
  static std::atomic<bool> configured[kMaxDevices] = {};
  return launch_tiles(fmoe_matmul_block128_hw_kernel<kPair>, configured, kHwThreads, HwCfg<kPair>::kSmemBytes, kPair ? 2 : 1, a, w, p,
                      grid, stream);
}

// Clusters of 1, 2, 4 and 8 CTAs that run side by side when a CTA has an SM to itself (a cluster does
// not straddle the groups that the SMs come in, so this is less than the SMs divided by its size).
struct ClusterRoom {
  int most[4];
};
template <int kNT, bool kBytes>
cudaError_t small_kernel_room(ClusterRoom* room) {
  static ClusterRoom known[kMaxDevices];
  static std::atomic<bool> configured[kMaxDevices] = {};
  auto kernel = fmoe_matmul_block128_small_kernel<kNT, kBytes>;
  int dev = 0;
  cudaGetDevice(&dev);
  const bool cached = dev >= 0 && dev < kMaxDevices;
  if (cached && configured[dev].load(std::memory_order_acquire)) {
    *room = known[dev];
    return cudaSuccess;
  }
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBsMostSmem);
  for (int i = 0; i < 4 && e == cudaSuccess; ++i) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1u << i;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(1024);
    cfg.blockDim = dim3(BlockSmallCfg<kNT>::kThreads);
    cfg.dynamicSmemBytes = kBsMostSmem;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&room->most[i], kernel, &cfg);
  }
  if (e == cudaSuccess && cached) {
    static std::mutex once;
    std::lock_guard<std::mutex> lock(once);
    if (!configured[dev].load(std::memory_order_relaxed)) known[dev] = *room;
    configured[dev].store(true, std::memory_order_release);
  }
  return e;
}

// Split K as far as all clusters run at once and every CTA keeps two blocks.
int small_log_split(int nt, int tiles, int kb, const ClusterRoom& room) {
  int log_split = 3;
  while (log_split > 0 && ((2 << log_split) > nt || tiles > room.most[log_split] || kb < (2 << log_split))) --log_split;
  return log_split;
}

// The room for clusters of the kernel with nt rows to a tile.
template <bool kBytes>
cudaError_t small_room(int nt, ClusterRoom* room) {
  switch (nt) {
    case 16: return small_kernel_room<16, kBytes>(room);
    case 32: return small_kernel_room<32, kBytes>(room);
    default: return small_kernel_room<128, kBytes>(room);
  }
}

template <int kNT, bool kBytes>
int run_small(const void* a, const void* w, BlockSmallParams p, int k, cudaStream_t stream) {
  using Cfg = BlockSmallCfg<kNT>;
  ClusterRoom room;
  FMOE_CUDA((small_kernel_room<kNT, kBytes>(&room)));
  CUtensorMap ta, tw;
  CUresult r = byte_map(&ta, a, p.m, k, kNT);
  if (r == CUDA_SUCCESS) r = byte_map(&tw, w, p.n, k, 128);
  if (r != CUDA_SUCCESS) return fail(FMOE_ERR_CUDA, "fmoe_matmul_block128: tensor map (driver code %d)", static_cast<int>(r));
  p.t_tiles = (p.m + kNT - 1) / kNT;
  const int tiles = p.t_tiles * ((p.n + 127) / 128);
  // A CTA alone on its SM takes the deep pipeline, two to an SM half of it each.
  const bool alone = tiles * p.split <= room.most[0] || Cfg::kTmemCols == 512;
  int stages = kBsMaxStages;
  while (stages > 2 && Cfg::smem_bytes(stages, p.split > 1) > (alone ? kBsMostSmem : 113 * 1024)) --stages;
  const int blocks_each = (p.kb + p.split - 1) / p.split;
  p.stages = stages < blocks_each ? stages : blocks_each;
  p.idesc = ptx::make_idesc(0u, 128, kNT);
  int smem = Cfg::smem_bytes(p.stages, p.split > 1);
  if (smem < Cfg::kMinSmem) smem = Cfg::kMinSmem;
  FMOE_CUDA(launch_pdl_cluster(fmoe_matmul_block128_small_kernel<kNT, kBytes>, dim3(tiles * p.split), dim3(Cfg::kThreads), smem,
                               p.split, stream, ta, tw, p));
  return FMOE_OK;
}

template <bool kBytes>
int run_small_nt(int nt, const void* a, const void* w, const BlockSmallParams& p, int k, cudaStream_t stream) {
  switch (nt) {
    case 16: return run_small<16, kBytes>(a, w, p, k, stream);
    case 32: return run_small<32, kBytes>(a, w, p, k, stream);
    default: return run_small<128, kBytes>(a, w, p, k, stream);
  }
}

// What a product runs on: the kernel, and for few rows the CTAs that share a tile's K blocks.
struct MatmulChoice {
  int kernel;      // kOneCta, kPairOfCtas, or the rows to a tile of the kernel for few rows
  int split;
};

// The kernel that is estimated to be done first: the one for few rows (16, 32 or 128 rows to a tile), or
// 128 x 256 tiles of a CTA (kOneCta), or 256 x 256 tiles of a pair of CTAs (kPairOfCtas).  An estimate
// is a fixed part (launch, set-up, the way of the first blocks, the result), with few rows one for each
// halving of K over a cluster, and a time for each K block of the longest CTA, in nanoseconds, fitted to
// measured times of 1 to 2048 rows times weights of 1024 x 1024 up to 18432 x 7168; the constants for few rows
// are those of f32 scales.  Over those sizes the choice between few rows and 128 x 256 is 1 % from the best
// on average with f32 scales and about 2 % with power-of-two scales; the worst single one found is 32 x 7744
// x 2048, 7.4 us where tiles of 16 rows take 5.7.  CTAs with 16 or 32 rows share an SM, which takes 1.6 times
// as many at the same time; with 128 rows there are whole rounds.  A pair's constants rest on two shapes: it
// starts 1.2 us later, but reads a third less from L2 and shared memory, which under the power limit is a
// higher clock: 8192 x 4096 x 7168 takes 191 to 194 us instead of 210 (power-of-two scales) and 237 instead of
// 253 (f32), 8192 x 1024 x 1024 12.2 instead of 11.6 and 16.1 instead of 14.8.
enum : int { kOneCta = 0, kPairOfCtas = 1 };
int choose_kernel(int64_t m, int n, int kb, bool hw, int sms, const ClusterRoom& room) {
  const int64_t n_tiles = (n + 127) / 128;
  const int tile_n = hw ? kHwTileN : kBmmTileN;
  const int64_t across = (n + tile_n - 1) / tile_n;
  auto rounds_of = [](int64_t tiles, int64_t at_once) { return static_cast<double>((tiles + at_once - 1) / at_once); };
  double best = (hw ? 4600.0 : 5000.0) + rounds_of((m + kBmmTileM - 1) / kBmmTileM * across, sms) * kb * (hw ? 330.0 : 440.0);
  int choice = kOneCta;
  const double pair = (hw ? 5700.0 : 6200.0) + rounds_of((m + 2 * kBmmTileM - 1) / (2 * kBmmTileM) * across, (sms + 1) / 2) * kb * (hw ? 305.0 : 418.0);
  if (sms > 1 && pair < best) { best = pair; choice = kPairOfCtas; }
  const struct { int nt; double fixed, halving, block, shared; } kinds[3] = {
      {16, 2000, 100, 300, 1.6}, {32, 3000, 200, 345, 1.6}, {128, 4800, 1200, 380, 1.0}};
  for (const auto& kind : kinds) {
    const int64_t tiles = (m + kind.nt - 1) / kind.nt * n_tiles;
    if (tiles > (int64_t{1} << 20)) continue;
    const int log_split = small_log_split(kind.nt, static_cast<int>(tiles), kb, room), split = 1 << log_split;
    const int64_t ctas = tiles * split;
    double rounds = kind.nt == 128 ? rounds_of(ctas, sms) : static_cast<double>(ctas) / (sms * kind.shared);
    if (rounds < 1.0) rounds = 1.0;
    const double t = kind.fixed + log_split * kind.halving + (kb + split - 1) / split * kind.block * rounds;
    if (t < best) { best = t; choice = kind.nt; }
  }
  return choice;
}

// For sizes that check_sizes has passed, on the current device.
template <bool kHw>
cudaError_t choose(int64_t m, int n, int kb, MatmulChoice* choice) {
  ClusterRoom room;
  cudaError_t e = small_room<kHw>(16, &room);
  if (e != cudaSuccess) return e;
  *choice = {choose_kernel(m, n, kb, kHw, device_sm_count(), room), 1};
  if (choice->kernel == kOneCta || choice->kernel == kPairOfCtas) return cudaSuccess;
  e = small_room<kHw>(choice->kernel, &room);
  const int64_t tiles = (m + choice->kernel - 1) / choice->kernel * ((n + 127) / 128);
  if (e == cudaSuccess) choice->split = 1 << small_log_split(choice->kernel, static_cast<int>(tiles), kb, room);
  return e;
}

int check_sizes(const char* name, int64_t m, int32_t n, int32_t k, int32_t quant) {
  if (quant != FMOE_QUANT_BLOCK128 && quant != FMOE_QUANT_BLOCK128_UE8M0)
    return fail(FMOE_ERR_INVALID_ARG, "%s: quant must be a block mode", name);
  if (m < 0 || n <= 0 || k <= 0)
    return fail(FMOE_ERR_INVALID_ARG, "%s: bad dimensions (m=%lld n=%d k=%d)", name, (long long)m, n, k);
  if (k % 128) return fail(FMOE_ERR_UNSUPPORTED, "%s: k must be a multiple of 128", name);
  if (m > 0x7fffff00LL || n > 0x7fffff00 || (m / kBmmTileM + 1) * (n / kBmmTileN + 1) > 0x7fffffffLL)
    return fail(FMOE_ERR_UNSUPPORTED, "%s: problem too large", name);
  return FMOE_OK;
}

}  // namespace

cudaError_t take_block_matmul_status(int32_t* code) {
  cudaError_t e = cudaMemcpyFromSymbol(code, g_bmm_status, sizeof(*code));
  const int32_t zero = 0;
  if (e == cudaSuccess && *code != 0) e = cudaMemcpyToSymbol(g_bmm_status, &zero, sizeof(zero));
  return e;
}
#ifdef FMOE_WAIT_LIMIT_SWITCH
cudaError_t set_block_matmul_wait_limit(int64_t cycles) {
  const long long limit = cycles;
  return cudaMemcpyToSymbol(ptx::g_wait_limit, &limit, sizeof(limit));
}
#endif
}  // namespace fmoe

extern "C" int fmoe_matmul_block128(const void* a, const void* a_scale, const void* w, const float* w_scale, int64_t m,
                                    int32_t n, int32_t k, int32_t quant, void* out, int32_t* status, void* stream) {
  using namespace fmoe;
  const int checked = check_sizes("fmoe_matmul_block128", m, n, k, quant);
  if (checked != FMOE_OK) return checked;
  if (m == 0) return FMOE_OK;
  if (!a || !a_scale || !w || !w_scale || !out)
    return fail(FMOE_ERR_INVALID_ARG, "fmoe_matmul_block128: a, a_scale, w, w_scale and out are required");
  auto misaligned = [](const void* p, uintptr_t mask) { return (reinterpret_cast<uintptr_t>(p) & mask) != 0; };
  if (misaligned(a, 15) || misaligned(w, 15) || misaligned(out, 15) || misaligned(a_scale, 3) || misaligned(w_scale, 3) ||
      misaligned(status, 3))
    return fail(FMOE_ERR_INVALID_ARG, "fmoe_matmul_block128: a, w and out must be 16-byte aligned, the scales and status 4-byte aligned");
  DeviceGuard guard(a);
  if (guard.rc() != FMOE_OK) return guard.rc();
  NvtxRange range("fmoe_matmul_block128");
  const int sms = device_sm_count();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool hw = quant == FMOE_QUANT_BLOCK128_UE8M0;
  MatmulChoice choice;
  FMOE_CUDA(hw ? choose<true>(m, n, k / 128, &choice) : choose<false>(m, n, k / 128, &choice));
  if (choice.kernel != kOneCta && choice.kernel != kPairOfCtas) {
    BlockSmallParams p{};
    p.a_scale = a_scale;
    p.w_scale = w_scale;
    p.m = static_cast<int>(m);
    p.n = n;
    p.kb = k / 128;
    p.split = choice.split;
    p.out = static_cast<__nv_bfloat16*>(out);
    p.status = status;
    return hw ? run_small_nt<true>(choice.kernel, a, w, p, k, s) : run_small_nt<false>(choice.kernel, a, w, p, k, s);
  }
  CUtensorMap ta, tw;
  CUresult r = byte_map(&ta, a, m, k, kBmmTileM);
  const int tile_n = hw ? kHwTileN : kBmmTileN;
  const bool pair = choice.kernel == kPairOfCtas;
  if (r == CUDA_SUCCESS) r = byte_map(&tw, w, n, k, !pair ? tile_n : hw ? HwCfg<true>::kWRows : BmmCfg<true>::kHalfRows);
  if (r != CUDA_SUCCESS) return fail(FMOE_ERR_CUDA, "fmoe_matmul_block128: tensor map (driver code %d)", static_cast<int>(r));
  BlockMatmulParams p{};
  p.a_scale = a_scale;
  p.w_scale = w_scale;
  p.m = static_cast<int>(m);
  p.n = n;
  p.kb = k / 128;
  const int tile_m = pair ? 2 * kBmmTileM : kBmmTileM;
  p.m_blocks = (p.m + tile_m - 1) / tile_m;
  p.n_blocks = (n + tile_n - 1) / tile_n;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.status = status;
  p.idesc = hw ? ptx::make_idesc_block_scaled(tile_m, kHwTileN) : ptx::make_idesc(0u, tile_m, kBmmTileN / 2);
  const int tiles = p.m_blocks * p.n_blocks;
  if (pair) {
    const int grid = 2 * (tiles < sms / 2 ? tiles : sms / 2);      // sms / 2 pairs run at once, or take turns: none waits for another
    FMOE_CUDA(hw ? launch_hw<true>(ta, tw, p, grid, s) : launch_f32<true>(ta, tw, p, grid, s));
  } else {
    const int grid = tiles < sms ? tiles : sms;
    FMOE_CUDA(hw ? launch_hw<false>(ta, tw, p, grid, s) : launch_f32<false>(ta, tw, p, grid, s));
  }
  return FMOE_OK;
}

extern "C" int fmoe_describe_matmul_block128(int64_t m, int32_t n, int32_t k, int32_t quant, fmoe_matmul_info_c* info) {
  using namespace fmoe;
  if (!info) return fail(FMOE_ERR_INVALID_ARG, "fmoe_describe_matmul_block128: info is required");
  *info = fmoe_matmul_info_c{};
  const int rc = check_sizes("fmoe_describe_matmul_block128", m, n, k, quant);
  if (rc != FMOE_OK || m == 0) return rc;
  MatmulChoice choice;
  FMOE_CUDA(quant == FMOE_QUANT_BLOCK128_UE8M0 ? choose<true>(m, n, k / 128, &choice) : choose<false>(m, n, k / 128, &choice));
  if (choice.kernel == kOneCta || choice.kernel == kPairOfCtas) {
    const bool pair = choice.kernel == kPairOfCtas;
    info->kernel = pair ? FMOE_MATMUL_CTA_PAIRS : FMOE_MATMUL_TILES;
    info->rows_per_tile = pair ? 2 * kBmmTileM : kBmmTileM;
    info->cols_per_tile = kBmmTileN;
  } else {
    info->kernel = FMOE_MATMUL_FEW_ROWS;
    info->rows_per_tile = choice.kernel;
    info->cols_per_tile = 128;
  }
  info->k_split = choice.split;
  return FMOE_OK;
}

extern "C" int fmoe_operator_status(int32_t device, int32_t* status_out) {
  using namespace fmoe;
  if (!status_out) return fail(FMOE_ERR_INVALID_ARG, "fmoe_operator_status: status_out is required");
  *status_out = 0;
  int before = 0;
  FMOE_CUDA(cudaGetDevice(&before));
  FMOE_CUDA(cudaSetDevice(device));
  int32_t code[2] = {0, 0};
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = take_grouped_status(&code[0]);
  if (e == cudaSuccess) e = take_block_matmul_status(&code[1]);
  cudaSetDevice(before);
  if (e != cudaSuccess) return fail(FMOE_ERR_CUDA, "fmoe_operator_status failed: %s", cudaGetErrorString(e));
  *status_out = code[0] ? code[0] : code[1];
  return FMOE_OK;
}

#ifdef FMOE_WAIT_LIMIT_SWITCH
// Limit of one wait in the operators' kernels, in clock cycles, on the current device.
extern "C" FMOE_API int fmoe_set_wait_limit(int64_t cycles) {
  using namespace fmoe;
  FMOE_CUDA(cudaDeviceSynchronize());
  FMOE_CUDA(set_grouped_wait_limit(cycles));
  FMOE_CUDA(set_block_matmul_wait_limit(cycles));
  return FMOE_OK;
}
#endif
