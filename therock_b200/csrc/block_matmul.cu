// Host side of the e4m3 product with block scales: checks, tensor maps, launch.
#include "block_matmul.cuh"

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

template <bool kBytes>
cudaError_t launch_promote(const CUtensorMap& a, const CUtensorMap& w, const BlockMatmulParams& p, int grid, cudaStream_t stream) {
  static bool configured[kMaxDevices] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices || !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(fmoe_matmul_block128_kernel<kBytes>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBmmSmemBytes);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < kMaxDevices) configured[dev] = true;
  }
  return launch_pdl(fmoe_matmul_block128_kernel<kBytes>, dim3(grid), dim3(kBmmThreads), kBmmSmemBytes, stream, a, w, p);
}

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
  p.idesc = ptx::make_idesc(0u, kBmmTileM, kBmmTileN / 2);
  const int tiles = p.m_blocks * p.n_blocks, sms = device_sm_count();
  const int grid = tiles < sms ? tiles : sms;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  FMOE_CUDA(quant == FMOE_QUANT_BLOCK128 ? launch_promote<false>(ta, tw, p, grid, s) : launch_promote<true>(ta, tw, p, grid, s));
  return FMOE_OK;
}
