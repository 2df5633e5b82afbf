// Host side of the e4m3 product with block scales: checks, tensor maps, launch.
#include "block_hw.cuh"
#include "block_small.cuh"

#include "host.cuh"
#include "internal.h"

namespace fmoe {
namespace {

constexpr int kMaxDevices = 64;

CUresult byte_map(CUtensorMap* tm, const void* base, int64_t rows, int cols, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(cols)};
  const uint32_t box[2] = {128, static_cast<uint32_t>(box_rows)};
  return encode_tensor_map(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box);
}

template <bool kHw>
cudaError_t launch_tiles(const CUtensorMap& a, const CUtensorMap& w, const BlockMatmulParams& p, int grid, cudaStream_t stream) {
  static bool configured[kMaxDevices] = {false};
  constexpr auto kernel = kHw ? fmoe_matmul_block128_hw_kernel : fmoe_matmul_block128_kernel;
  constexpr int kSmem = kHw ? kHwSmemBytes : kBmmSmemBytes;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices || !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < kMaxDevices) configured[dev] = true;
  }
  return launch_pdl(kernel, dim3(grid), dim3(kBmmThreads), kSmem, stream, a, w, p);
}

template <int kNT, bool kBytes>
int run_small(const void* a, const void* w, BlockSmallParams p, int k, int sms, cudaStream_t stream) {
  using Cfg = BlockSmallCfg<kNT>;
  CUtensorMap ta, tw;
  CUresult r = byte_map(&ta, a, p.m, k, kNT);
  if (r == CUDA_SUCCESS) r = byte_map(&tw, w, p.n, k, 128);
  if (r != CUDA_SUCCESS) return fail(FMOE_ERR_CUDA, "fmoe_matmul_block128: tensor map (driver code %d)", static_cast<int>(r));
  p.t_tiles = (p.m + kNT - 1) / kNT;
  const int tiles = p.t_tiles * ((p.n + 127) / 128);
  // Split K while the CTAs still fit the GPU side by side and each keeps two blocks.
  p.split = 1;
  while (p.split < 8 && 2 * p.split <= kNT / 2 && tiles * p.split * 2 <= sms && p.kb >= 4 * p.split) p.split *= 2;
  // A CTA alone on its SM takes the deep pipeline, two to an SM half of it each.
  const int room = tiles * p.split <= sms || Cfg::kTmemCols == 512 ? 220 * 1024 : 113 * 1024;
  int stages = kBsMaxStages;
  while (stages > 2 && Cfg::smem_bytes(stages, p.split > 1) > room) --stages;
  const int blocks_each = (p.kb + p.split - 1) / p.split;
  p.stages = stages < blocks_each ? stages : blocks_each;
  p.idesc = ptx::make_idesc(0u, 128, kNT);
  static bool configured[kMaxDevices] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  auto kernel = fmoe_matmul_block128_small_kernel<kNT, kBytes>;
  if (dev < 0 || dev >= kMaxDevices || !configured[dev]) {
    FMOE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024));
    if (dev >= 0 && dev < kMaxDevices) configured[dev] = true;
  }
  int smem = Cfg::smem_bytes(p.stages, p.split > 1);
  if (smem < Cfg::kMinSmem) smem = Cfg::kMinSmem;
  FMOE_CUDA(launch_pdl_cluster(kernel, dim3(tiles * p.split), dim3(Cfg::kThreads), smem, p.split, stream, ta, tw, p));
  return FMOE_OK;
}

template <bool kBytes>
int run_small_nt(int nt, const void* a, const void* w, const BlockSmallParams& p, int k, int sms, cudaStream_t stream) {
  switch (nt) {
    case 16: return run_small<16, kBytes>(a, w, p, k, sms, stream);
    case 32: return run_small<32, kBytes>(a, w, p, k, sms, stream);
    case 64: return run_small<64, kBytes>(a, w, p, k, sms, stream);
    default: return run_small<128, kBytes>(a, w, p, k, sms, stream);
  }
}

// Rows per tile of the kernel for few rows, 0 for the kernel with 128 x 256 tiles.
int small_rows(int64_t m) { return m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : m <= 256 ? 128 : 0; }

}  // namespace
}  // namespace fmoe

extern "C" int fmoe_matmul_block128(const void* a, const void* a_scale, const void* w, const float* w_scale, int64_t m,
                                    int32_t n, int32_t k, int32_t quant, void* out, int32_t* status, void* stream) {
  using namespace fmoe;
  if (quant != FMOE_QUANT_BLOCK128 && quant != FMOE_QUANT_BLOCK128_UE8M0)
    return fail(FMOE_ERR_INVALID_ARG, "fmoe_matmul_block128: quant must be a block mode");
  if (m < 0 || n <= 0 || k <= 0)
    return fail(FMOE_ERR_INVALID_ARG, "fmoe_matmul_block128: bad dimensions (m=%lld n=%d k=%d)", (long long)m, n, k);
  if (k % 128) return fail(FMOE_ERR_UNSUPPORTED, "fmoe_matmul_block128: k must be a multiple of 128");
  if (m > 0x7fffff00LL || (m / kBmmTileM + 1) * (n / kBmmTileN + 1) > 0x7fffffffLL)
    return fail(FMOE_ERR_UNSUPPORTED, "fmoe_matmul_block128: problem too large");
  if (m == 0) return FMOE_OK;
  if (!a || !a_scale || !w || !w_scale || !out)
    return fail(FMOE_ERR_INVALID_ARG, "fmoe_matmul_block128: a, a_scale, w, w_scale and out are required");
  auto misaligned = [](const void* p, uintptr_t mask) { return (reinterpret_cast<uintptr_t>(p) & mask) != 0; };
  if (misaligned(a, 15) || misaligned(w, 15) || misaligned(out, 15) || misaligned(a_scale, 3) || misaligned(w_scale, 3))
    return fail(FMOE_ERR_INVALID_ARG, "fmoe_matmul_block128: a, w and out must be 16-byte aligned, the scales 4-byte aligned");
  DeviceGuard guard(a);
  if (guard.rc() != FMOE_OK) return guard.rc();
  NvtxRange range("fmoe_matmul_block128");
  const int sms = device_sm_count();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (const int nt = small_rows(m)) {
    BlockSmallParams p{};
    p.a_scale = a_scale;
    p.w_scale = w_scale;
    p.m = static_cast<int>(m);
    p.n = n;
    p.kb = k / 128;
    p.out = static_cast<__nv_bfloat16*>(out);
    p.status = status;
    return quant == FMOE_QUANT_BLOCK128 ? run_small_nt<false>(nt, a, w, p, k, sms, s) : run_small_nt<true>(nt, a, w, p, k, sms, s);
  }
  CUtensorMap ta, tw;
  CUresult r = byte_map(&ta, a, m, k, kBmmTileM);
  if (r == CUDA_SUCCESS) r = byte_map(&tw, w, n, k, kBmmTileN);
  if (r != CUDA_SUCCESS) return fail(FMOE_ERR_CUDA, "fmoe_matmul_block128: tensor map (driver code %d)", static_cast<int>(r));
  BlockMatmulParams p{};
  p.a_scale = a_scale;
  p.w_scale = w_scale;
  p.m = static_cast<int>(m);
  p.n = n;
  p.kb = k / 128;
  p.m_blocks = (p.m + kBmmTileM - 1) / kBmmTileM;
  p.n_blocks = (n + kBmmTileN - 1) / kBmmTileN;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.status = status;
  const bool hw = quant == FMOE_QUANT_BLOCK128_UE8M0;
  p.idesc = hw ? ptx::make_idesc_block_scaled(kBmmTileM, kBmmTileN) : ptx::make_idesc(0u, kBmmTileM, kBmmTileN / 2);
  const int tiles = p.m_blocks * p.n_blocks;
  const int grid = tiles < sms ? tiles : sms;
  FMOE_CUDA(hw ? launch_tiles<true>(ta, tw, p, grid, s) : launch_tiles<false>(ta, tw, p, grid, s));
  return FMOE_OK;
}
