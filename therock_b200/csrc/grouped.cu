// Host side of the products grouped by expert: checks, tensor maps, launches.
#include <atomic>

#include "grouped.cuh"

#include "host.cuh"
#include "internal.h"

namespace fmoe {
namespace {

constexpr int kMaxDevices = 64;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

int check_grouped(const char* name, const int32_t* offsets, int64_t rows, int32_t groups, int32_t n, int32_t k, int32_t dtype,
                  const int32_t* status) {
  if (!offsets) return fail(FMOE_ERR_INVALID_ARG, "%s: offsets are required", name);
  if (!aligned4(offsets) || !aligned4(status))
    return fail(FMOE_ERR_INVALID_ARG, "%s: offsets and status must be 4-byte aligned", name);
  if (rows < 0 || groups <= 0 || n <= 0 || k <= 0)
    return fail(FMOE_ERR_INVALID_ARG, "%s: bad dimensions (rows=%lld groups=%d n=%d k=%d)", name, (long long)rows, groups, n, k);
  if (dtype != FMOE_BF16 && dtype != FMOE_F16) return fail(FMOE_ERR_UNSUPPORTED, "%s: bf16 and f16 only", name);
  if (groups > kGrpMaxGroups) return fail(FMOE_ERR_UNSUPPORTED, "%s: at most %d groups", name, kGrpMaxGroups);
  if (n % 8 || k % 8) return fail(FMOE_ERR_UNSUPPORTED, "%s: n and k must be multiples of 8", name);
  // Row, column and tile numbers are 32-bit: a size plus a tile has to fit, and a group's rows plus the number of
  // its pieces of 256.
  const int64_t wide = (n > k ? n : k) / kGrpTile + 1;
  if (rows > 0x7f000000LL || n > 0x7fffff00 || k > 0x7fffff00 || (rows / kGrpTile + groups + 1) * wide > 0x7fffffffLL ||
      static_cast<int64_t>(groups) * (n / kGrpTile + 1) * (k / kGrpTile + 1) > 0x7fffffffLL)
    return fail(FMOE_ERR_UNSUPPORTED, "%s: problem too large", name);
  return FMOE_OK;
}

CUtensorMapDataType map_type(int dtype) {
  return dtype == FMOE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// Boxes of `box_rows` rows x 64 elements of a [rows, cols] matrix.
CUresult row_map(CUtensorMap* tm, int dtype, const void* base, int64_t rows, int cols, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(cols) * 2};
  const uint32_t box[2] = {kGrpStageK, static_cast<uint32_t>(box_rows)};
  return encode_tensor_map(tm, map_type(dtype), 2, base, dims, strides, box);
}
// The same of one group of w [groups, n, k]: rows behind a group's n are zeros, not the next group's.
CUresult weight_map(CUtensorMap* tm, int dtype, const void* base, int groups, int n, int k, int box_rows) {
  const uint64_t dims[3] = {static_cast<uint64_t>(k), static_cast<uint64_t>(n), static_cast<uint64_t>(groups)};
  const uint64_t strides[2] = {static_cast<uint64_t>(k) * 2, static_cast<uint64_t>(k) * n * 2};
  const uint32_t box[3] = {kGrpStageK, static_cast<uint32_t>(box_rows), 1};
  return encode_tensor_map(tm, map_type(dtype), 3, base, dims, strides, box);
}

template <typename Kernel, typename... Args>
cudaError_t launch_grouped(Kernel kernel, std::atomic<bool> (&configured)[kMaxDevices], int pairs, int threads, int smem, cudaStream_t stream,
                           const Args&... args) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices || !configured[dev].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < kMaxDevices) configured[dev].store(true, std::memory_order_release);
  }
  return launch_pdl(kernel, dim3(2 * pairs), dim3(threads), smem, stream, args...);
}
template <bool kBf16, bool kMn>
cudaError_t launch_rows(const CUtensorMap& w, const RowMaps& x, const GroupedParams& p, int pairs, cudaStream_t stream) {
  static std::atomic<bool> configured[kMaxDevices] = {};
  return launch_grouped(fmoe_grouped_rows_kernel<kBf16, kMn>, configured, pairs, kGrpThreads, kGrpSmemBytes, stream, w, x, p);
}
template <bool kBf16>
cudaError_t launch_wgrad(const CUtensorMap& dy, const CUtensorMap& x, const CUtensorMap& dw, const GroupedParams& p, int pairs,
                         cudaStream_t stream) {
  static std::atomic<bool> configured[kMaxDevices] = {};
  return launch_grouped(fmoe_grouped_wgrad_kernel<kBf16>, configured, pairs, kWgThreads, kWgSmemBytes, stream, dy, x, dw, p);
}

int pairs_for(int64_t tiles) {
  const int64_t most = device_sm_count() / 2;
  return static_cast<int>(tiles < 1 ? 1 : (tiles < most ? tiles : most));
}

}  // namespace

cudaError_t take_grouped_status(int32_t* code) {
  cudaError_t e = cudaMemcpyFromSymbol(code, g_grouped_status, sizeof(*code));
  const int32_t zero = 0;
  if (e == cudaSuccess && *code != 0) e = cudaMemcpyToSymbol(g_grouped_status, &zero, sizeof(zero));
  return e;
}
#ifdef FMOE_WAIT_LIMIT_SWITCH
cudaError_t set_grouped_wait_limit(int64_t cycles) {
  const long long limit = cycles;
  return cudaMemcpyToSymbol(ptx::g_wait_limit, &limit, sizeof(limit));
}
#endif
}  // namespace fmoe

extern "C" int fmoe_grouped_matmul(const void* x, const void* w, const int32_t* offsets, int64_t rows, int32_t groups,
                                   int32_t n, int32_t k, int32_t dtype, int32_t transpose_w, void* out, int32_t* status,
                                   void* stream_v) {
  using namespace fmoe;
  int rc = check_grouped("fmoe_grouped_matmul", offsets, rows, groups, n, k, dtype, status);
  if (rc != FMOE_OK) return rc;
  if (transpose_w != 0 && transpose_w != 1) return fail(FMOE_ERR_INVALID_ARG, "fmoe_grouped_matmul: transpose_w must be 0 or 1");
  if (rows == 0) return FMOE_OK;
  if (!x || !w || !out) return fail(FMOE_ERR_INVALID_ARG, "fmoe_grouped_matmul: x, w and out are required");
  if (!aligned16(x) || !aligned16(w) || !aligned16(out))
    return fail(FMOE_ERR_INVALID_ARG, "fmoe_grouped_matmul: x, w and out must be 16-byte aligned");
  DeviceGuard guard(x);
  if (guard.rc() != FMOE_OK) return guard.rc();
  NvtxRange range("fmoe_grouped_matmul");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  const int reduce = transpose_w ? n : k, cols = transpose_w ? k : n;
  CUtensorMap tw;
  RowMaps tx;
  CUresult r = weight_map(&tw, dtype, w, groups, n, k, transpose_w ? kGrpStageK : 128);
  for (int i = 0; i < 4 && r == CUDA_SUCCESS; ++i) r = row_map(&tx.m[i], dtype, x, rows, reduce, 128 >> i);
  if (r != CUDA_SUCCESS) return fail(FMOE_ERR_CUDA, "fmoe_grouped_matmul: tensor map (driver code %d)", static_cast<int>(r));
  GroupedParams p{};
  p.offsets = offsets;
  p.groups = groups;
  p.rows = static_cast<int>(rows);
  p.m_blocks = (cols + kGrpTile - 1) / kGrpTile;
  p.k_iters = (reduce + kGrpStageK - 1) / kGrpStageK;
  p.n = cols;
  p.out = static_cast<uint16_t*>(out);
  p.status = status;
  p.idesc = ptx::make_idesc(dtype == FMOE_BF16 ? 1u : 0u, 256, 0) | (transpose_w ? ptx::kIdescAMnMajor : 0u);
  const int pairs = pairs_for((rows / kGrpTile + (rows < groups ? rows : groups)) * p.m_blocks);
  if (dtype == FMOE_BF16)
    FMOE_CUDA(transpose_w ? (launch_rows<true, true>(tw, tx, p, pairs, stream)) : (launch_rows<true, false>(tw, tx, p, pairs, stream)));
  else
    FMOE_CUDA(transpose_w ? (launch_rows<false, true>(tw, tx, p, pairs, stream)) : (launch_rows<false, false>(tw, tx, p, pairs, stream)));
  return FMOE_OK;
}

extern "C" int fmoe_grouped_matmul_wgrad(const void* dy, const void* x, const int32_t* offsets, int64_t rows, int32_t groups,
                                         int32_t n, int32_t k, int32_t dtype, void* dw, int32_t* status, void* stream_v) {
  using namespace fmoe;
  int rc = check_grouped("fmoe_grouped_matmul_wgrad", offsets, rows, groups, n, k, dtype, status);
  if (rc != FMOE_OK) return rc;
  if (!dw || (rows > 0 && (!dy || !x))) return fail(FMOE_ERR_INVALID_ARG, "fmoe_grouped_matmul_wgrad: dy, x and dw are required");
  if (!aligned16(dy) || !aligned16(x) || !aligned16(dw))
    return fail(FMOE_ERR_INVALID_ARG, "fmoe_grouped_matmul_wgrad: dy, x and dw must be 16-byte aligned");
  DeviceGuard guard(dw);
  if (guard.rc() != FMOE_OK) return guard.rc();
  NvtxRange range("fmoe_grouped_matmul_wgrad");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (rows == 0) {      // no tensor map can describe a matrix without rows
    FMOE_CUDA(cudaMemsetAsync(dw, 0, static_cast<size_t>(groups) * n * k * 2, stream));
    return FMOE_OK;
  }
  CUtensorMap tdy, tx, tdw;
  CUresult r = row_map(&tdy, dtype, dy, rows, n, kGrpStageK);
  if (r == CUDA_SUCCESS) r = row_map(&tx, dtype, x, rows, k, kGrpStageK);
  if (r == CUDA_SUCCESS) r = weight_map(&tdw, dtype, dw, groups, n, k, 32);
  if (r != CUDA_SUCCESS) return fail(FMOE_ERR_CUDA, "fmoe_grouped_matmul_wgrad: tensor map (driver code %d)", static_cast<int>(r));
  GroupedParams p{};
  p.offsets = offsets;
  p.groups = groups;
  p.rows = static_cast<int>(rows);
  p.m_blocks = (n + kGrpTile - 1) / kGrpTile;
  p.k_blocks = (k + kGrpTile - 1) / kGrpTile;
  p.n = n;
  p.k = k;
  p.out = static_cast<uint16_t*>(dw);
  p.status = status;
  p.idesc = ptx::make_idesc(dtype == FMOE_BF16 ? 1u : 0u, 256, 256) | ptx::kIdescAMnMajor | ptx::kIdescBMnMajor;
  const int pairs = pairs_for(static_cast<int64_t>(groups) * p.m_blocks * p.k_blocks);
  FMOE_CUDA(dtype == FMOE_BF16 ? launch_wgrad<true>(tdy, tx, tdw, p, pairs, stream) : launch_wgrad<false>(tdy, tx, tdw, p, pairs, stream));
  return FMOE_OK;
}
