// C ABI of the routed row movements and the block quantiser (include/magi_swiglu.h): argument checks and launches.
// Device code lives in routed_kernels.cuh.
#include "host_common.hpp"
#include "routed_kernels.cuh"

namespace magi {

// Threads of a block over one row's 16-byte pieces (x) and several rows (y), and how many blocks cover a row.
struct RowGrid {
  dim3 block;
  unsigned grid;
  int col_chunks;
};
static int row_grid(int64_t rows, int64_t pieces, RowGrid* g) {
  const int64_t wide = (pieces + 31) / 32 * 32;
  const unsigned bx = (unsigned)(wide < 256 ? wide : 256), by = 256 / bx;
  const int64_t chunks = (pieces + bx - 1) / bx, blocks = (rows + by - 1) / by * chunks;
  if (blocks > 0x7fffffffLL) return fail(MAGI_SWIGLU_ERR_SHAPE, "too many rows x columns for one launch");
  g->block = dim3(bx, by);
  g->grid = (unsigned)blocks;
  g->col_chunks = (int)chunks;
  return 0;
}

static int check_rows(int64_t T, int64_t k, int64_t H, int64_t ld, int multiple) {
  if (T < 0 || k < 1 || H < 1 || T > 0x7fffffffLL / k)
    return fail(MAGI_SWIGLU_ERR_SHAPE, "T=%lld, k=%lld, H=%lld out of range (T * k < 2^31)", (long long)T, (long long)k,
                (long long)H);
  if (H % multiple) return fail(MAGI_SWIGLU_ERR_SHAPE, "the row length %lld must be a multiple of %d", (long long)H, multiple);
  if (H > 0x7fffffffLL || ld < H) return fail(MAGI_SWIGLU_ERR_SHAPE, "row stride %lld too small for %lld columns", (long long)ld, (long long)H);
  if (ld % 8) return fail(MAGI_SWIGLU_ERR_ALIGN, "row strides must be multiples of 8 elements");
  return 0;
}
static bool unaligned(const void* a, const void* b = nullptr, const void* c = nullptr) {
  return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15u) != 0;
}

constexpr int kSortSmemMax = (32 + 3) * (kMaxExperts + 1) * (int)sizeof(int);

// The largest cluster the sort may use on `device` (the current device): 16 CTAs where the GPU schedules that many
// together at the kernel's largest size, else 8; 0 if not even those.  Looked up once per device.
static int sort_cluster(int device) {
  static int known[kMaxDevices];
  std::lock_guard<std::mutex> lock(g_dev_mutex);
  if (known[device]) return known[device];
  cudaFuncSetAttribute(expert_sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  for (int ctas = kSortCtas; ctas >= 8; ctas -= 8) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(1024);
    cfg.dynamicSmemBytes = kSortSmemMax;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, expert_sort_kernel, &cfg) == cudaSuccess && n > 0) return known[device] = ctas;
    cudaGetLastError();
  }
  return 0;
}

static int quantize(const void* x, const int32_t* row_slot, const int32_t* slot_row, void* codes, float* scales, int64_t T,
                    int64_t k, int64_t K, int64_t ldx, int device, void* stream) {
  if (int rc = check_rows(T, k, K, ldx, 16)) return rc;
  if (T == 0) return 0;
  if (!x || !codes || !scales) return fail(MAGI_SWIGLU_ERR_NULL, "null pointer argument");
  if (unaligned(x, codes)) return fail(MAGI_SWIGLU_ERR_ALIGN, "x and codes must be 16-byte aligned");
  const DeviceInfo* di = nullptr;
  if (int rc = require_b200(device, &di)) return rc;
  RowGrid g;
  if (int rc = row_grid(T, K / 16, &g)) return rc;
  DeviceGuard guard;
  cudaError_t e = guard.set(device);
  if (e != cudaSuccess) return fail_cuda(e, "cudaSetDevice");
  e = launch(quantize_fp8_block_kernel, dim3(g.grid), g.block, 0, static_cast<cudaStream_t>(stream), 1u, true,
             static_cast<const uint4*>(x), ldx / 8, row_slot, slot_row, static_cast<uint4*>(codes), scales, T,
             (int)k, (int)(K / 16), g.col_chunks, (int)((K + 127) / 128));
  return e == cudaSuccess ? 0 : fail_cuda(e, "launch of quantize_fp8_block_kernel");
}

}  // namespace magi

using namespace magi;

extern "C" {

int magi_swiglu_expert_sort(const void* ids, int ids_64bit, int64_t slots, int num_experts, int32_t* row_slot,
                            int32_t* slot_row, int32_t* offsets, int device, void* cuda_stream) {
  g_err[0] = 0;
  if (slots < 0 || slots > 0x3fffffffLL) return fail(MAGI_SWIGLU_ERR_SHAPE, "slots=%lld out of range [0, 2^30)", (long long)slots);
  if (num_experts < 1 || num_experts > kMaxExperts)
    return fail(MAGI_SWIGLU_ERR_SHAPE, "num_experts=%d out of range [1, %d]", num_experts, kMaxExperts);
  if (!offsets || (slots > 0 && (!ids || !row_slot || !slot_row))) return fail(MAGI_SWIGLU_ERR_NULL, "null pointer argument");
  if (((uintptr_t)ids & (ids_64bit ? 7u : 3u)) || (((uintptr_t)row_slot | (uintptr_t)slot_row | (uintptr_t)offsets) & 3u))
    return fail(MAGI_SWIGLU_ERR_ALIGN, "index arrays must be aligned to their element size");
  const DeviceInfo* di = nullptr;
  if (int rc = require_b200(device, &di)) return rc;
  DeviceGuard guard;
  cudaError_t e = guard.set(device);
  if (e != cudaSuccess) return fail_cuda(e, "cudaSetDevice");
  static int smem_set[kMaxDevices];
  e = allow_smem_once(expert_sort_kernel, kSortSmemMax, device, smem_set);
  if (e != cudaSuccess) return fail_cuda(e, "cudaFuncSetAttribute(MaxDynamicSharedMemorySize)");
  // A warp takes 128 slots before another joins, and the warps are spread over as many CTAs as a cluster has: votes and
  // scattered stores share an SM's units (16384 slots of 8 experts: 2 CTAs of 32 warps 12.1 us, 8 of 16 warps 4.4 us; 32792
  // slots of 128: 8 CTAs 12.0 us, 16 CTAs 7.8 us).  Up to 1024 slots one CTA does without the cluster's barriers.
  const int64_t all_warps = (slots + 127) / 128;
  int ctas = 1;
  if (all_warps > 8) {
    const int most = sort_cluster(device);
    if (most <= 0) return fail(MAGI_SWIGLU_ERR_DEVICE, "expert_sort_kernel cannot run as a cluster on device %d", device);
    ctas = all_warps <= 64 ? 8 : most;
    if (ctas > most) ctas = most;
  }
  int warps = (int)((all_warps + ctas - 1) / ctas);
  warps = warps < 4 ? 4 : (warps > 32 ? 32 : warps);
  const size_t smem = (size_t)(warps + 3) * (num_experts + 1) * sizeof(int);
  e = launch(expert_sort_kernel, dim3((unsigned)ctas), dim3((unsigned)warps * 32), smem,
             static_cast<cudaStream_t>(cuda_stream), (unsigned)ctas, true, ids, ids_64bit, (int)slots, num_experts,
             (int*)row_slot, (int*)slot_row, (int*)offsets, ctas);
  return e == cudaSuccess ? 0 : fail_cuda(e, "launch of expert_sort_kernel");
}

int magi_swiglu_expert_gather_bf16(const void* x, const int32_t* row_slot, const int32_t* slot_row, void* xs, int64_t T,
                                   int64_t k, int64_t H, int64_t ldx, int device, void* cuda_stream) {
  g_err[0] = 0;
  if (int rc = check_rows(T, k, H, ldx, 8)) return rc;
  if (T == 0) return 0;
  if (!x || !row_slot || !slot_row || !xs) return fail(MAGI_SWIGLU_ERR_NULL, "null pointer argument");
  if (unaligned(x, xs)) return fail(MAGI_SWIGLU_ERR_ALIGN, "x and xs must be 16-byte aligned");
  const DeviceInfo* di = nullptr;
  if (int rc = require_b200(device, &di)) return rc;
  RowGrid g;
  if (int rc = row_grid(T, H / 8, &g)) return rc;
  DeviceGuard guard;
  cudaError_t e = guard.set(device);
  if (e != cudaSuccess) return fail_cuda(e, "cudaSetDevice");
  e = launch(expert_gather_kernel, dim3(g.grid), g.block, 0, static_cast<cudaStream_t>(cuda_stream), 1u, true,
             static_cast<const uint4*>(x), ldx / 8, row_slot, slot_row, static_cast<uint4*>(xs), T, (int)k,
             (int)(H / 8), g.col_chunks);
  return e == cudaSuccess ? 0 : fail_cuda(e, "launch of expert_gather_kernel");
}

int magi_swiglu_expert_combine_bf16(const void* y, const float* weights, const int32_t* slot_row, void* out, int64_t T,
                                    int64_t k, int64_t H, int64_t ldy, int device, void* cuda_stream) {
  g_err[0] = 0;
  if (int rc = check_rows(T, k, H, ldy, 8)) return rc;
  if (T == 0) return 0;
  if (!y || !slot_row || !out) return fail(MAGI_SWIGLU_ERR_NULL, "null pointer argument");
  if (unaligned(y, out)) return fail(MAGI_SWIGLU_ERR_ALIGN, "y and out must be 16-byte aligned");
  const DeviceInfo* di = nullptr;
  if (int rc = require_b200(device, &di)) return rc;
  // up to eight loads in flight per thread, split between the token's rows and column pieces
  const int pieces = k <= 2 ? 4 : (k <= 4 ? 2 : 1);
  RowGrid g;
  if (int rc = row_grid(T, (H / 8 + pieces - 1) / pieces, &g)) return rc;
  DeviceGuard guard;
  cudaError_t e = guard.set(device);
  if (e != cudaSuccess) return fail_cuda(e, "cudaSetDevice");
  auto kernel = k <= 1 ? expert_combine_kernel<1, 4> : k <= 2 ? expert_combine_kernel<2, 4>
                : k <= 4 ? expert_combine_kernel<4, 2> : expert_combine_kernel<8, 1>;
  e = launch(kernel, dim3(g.grid), g.block, 0, static_cast<cudaStream_t>(cuda_stream), 1u, true,
             static_cast<const uint4*>(y), ldy / 8, weights, slot_row, static_cast<uint4*>(out), T, (int)k,
             (int)(H / 8), g.col_chunks);
  return e == cudaSuccess ? 0 : fail_cuda(e, "launch of expert_combine_kernel");
}

int magi_swiglu_expert_combine_backward_bf16(const void* dout, const void* y, const float* weights, const int32_t* row_slot,
                                             const int32_t* slot_row, void* dy, float* dw, int64_t T, int64_t k, int64_t H,
                                             int64_t lddout, int64_t ldy, int device, void* cuda_stream) {
  g_err[0] = 0;
  if (int rc = check_rows(T, k, H, lddout, 8)) return rc;
  if (dw)
    if (int rc = check_rows(T, k, H, ldy, 8)) return rc;
  if (T == 0 || (!dy && !dw)) return 0;
  if (!dout || !slot_row || (dy && (!weights || !row_slot)) || (dw && !y)) return fail(MAGI_SWIGLU_ERR_NULL, "null pointer argument");
  if (unaligned(dout, dw ? y : nullptr, dy)) return fail(MAGI_SWIGLU_ERR_ALIGN, "dout, y and dy must be 16-byte aligned");
  const DeviceInfo* di = nullptr;
  if (int rc = require_b200(device, &di)) return rc;
  DeviceGuard guard;
  cudaError_t e = guard.set(device);
  if (e != cudaSuccess) return fail_cuda(e, "cudaSetDevice");
  // One warp walks a whole token when there are enough tokens to fill the GPU (8 warps a block, 4 blocks an SM); few
  // tokens get up to eight warps each, as far as the row has pieces for them.
  int token_warps = 1;
  while (token_warps < 8 && T * token_warps < (int64_t)di->sm_count * 32 && H / 8 > token_warps * 32) token_warps *= 2;
  const int64_t blocks = (T + 8 / token_warps - 1) / (8 / token_warps);
  e = launch(expert_combine_backward_kernel, dim3((unsigned)blocks), dim3(256), 0,
             static_cast<cudaStream_t>(cuda_stream), 1u, true, static_cast<const uint4*>(dout), lddout / 8,
             static_cast<const uint4*>(y), ldy / 8, weights, row_slot, slot_row, static_cast<uint4*>(dy), dw, T,
             (int)k, (int)(H / 8), token_warps);
  return e == cudaSuccess ? 0 : fail_cuda(e, "launch of expert_combine_backward_kernel");
}

int magi_swiglu_quantize_fp8_block(const void* x, void* codes, float* scales, int64_t M, int64_t K, int64_t ldx, int device,
                                   void* cuda_stream) {
  g_err[0] = 0;
  return quantize(x, nullptr, nullptr, codes, scales, M, 1, K, ldx, device, cuda_stream);
}

int magi_swiglu_expert_gather_fp8_block(const void* x, const int32_t* row_slot, const int32_t* slot_row, void* codes,
                                        float* scales, int64_t T, int64_t k, int64_t K, int64_t ldx, int device,
                                        void* cuda_stream) {
  g_err[0] = 0;
  if (T > 0 && (!row_slot || !slot_row)) return fail(MAGI_SWIGLU_ERR_NULL, "null pointer argument");
  return quantize(x, row_slot, slot_row, codes, scales, T, k, K, ldx, device, cuda_stream);
}

}  // extern "C"
