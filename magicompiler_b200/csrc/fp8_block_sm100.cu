// C ABI of the block-scaled fp8 products (include/magi_swiglu.h): argument checks, tile choice, tensor maps, launches.
// Device code lives in fp8_block_kernels.cuh.
#include <cmath>
#include <cstring>

#include "fp8_block_kernels.cuh"
#include "host_common.hpp"

namespace magi {

// Read and clear this translation unit's watchdog word (the device is current and idle).
cudaError_t fp8_block_watchdog(unsigned int out[4]) {
  cudaError_t e = cudaMemcpyFromSymbol(out, fp8::g_fp8_watchdog, 4 * sizeof(unsigned int));
  if (e == cudaSuccess && out[0] != 0) {
    const unsigned int zero[4] = {0, 0, 0, 0};
    e = cudaMemcpyToSymbol(fp8::g_fp8_watchdog, zero, sizeof(zero));
  }
  return e;
}

namespace fp8 {

static int encode_bytes_map(const void* ptr, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                            const cuuint32_t* box, CUtensorMap* tm, const char* what) {
  EncodeTiledFn enc = tensor_map_encoder();
  if (!enc) return fail(MAGI_SWIGLU_ERR_DRIVER, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, (cuuint32_t)rank, const_cast<void*>(ptr), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MAGI_SWIGLU_ERR_DRIVER, "tensor map for %s rejected by the driver (CUresult %d)", what, (int)r);
  return 0;
}

struct Problem {
  const void* a;
  const void* b;
  long long lda;
  int64_t M, N, K;
  int halves;
  bool routed;  // rows belong to experts (offsets)
  Args args;
};

// Which kernel runs: the stream kernel with `tok` rows a tile, or (tok 0) tiles of `ctas` CTAs; `splits` CTAs or pairs of a
// cluster share a tile's K blocks.
struct Form {
  int tok, ctas, splits;
};

// Row groups of `rows` rows: every expert adds at most one partial group.
static int64_t most_groups(const Problem& p, int rows) {
  return p.routed ? p.M / rows + (p.M < p.args.E + 1 ? p.M : p.args.E + 1) : (p.M + rows - 1) / rows;
}
// What to expect of them: experts' shares are uneven, and an exponentially distributed share of mean s needs 1 / (1 -
// exp(-rows / s)) groups on average (one for a small share, s / rows + 1/2 for a large one).
static double expected_groups(const Problem& p, int rows) {
  if (!p.routed) return (double)((p.M + rows - 1) / rows);
  const double used = (double)(p.M < p.args.E ? p.M : p.args.E);
  return used / (1.0 - exp(-rows * used / (double)p.M));
}
// Rounds of `workers` at a time; an expected count may miss by a few per cent, which must not make a round.
static double rounds_of(const Problem& p, double tiles, double workers) {
  return p.routed ? fmax(1.0, ceil(0.97 * tiles / workers)) : ceil(tiles / workers);
}

template <int kHalves, int kTok>
static int launch_stream(const Problem& p, int device, int splits, cudaStream_t stream) {
  constexpr int kStage = kHalves * kWTile + kTok * kBlk;
  // Two CTAs an SM, and no room beside one for a CTA of the bf16 kernels, which take at least 120 KB and all of tensor
  // memory: two clusters whose CTAs wait for each other's tensor memory on two SMs would wait for good.
  constexpr int kSmem = 108 * 1024;
  constexpr int kFit = (kSmem - 1024) / kStage;
  constexpr int kStages = kFit < kMaxStages ? kFit : kMaxStages;
  static_assert(kStages >= 2 && kStages * kStage >= kTok * kHalves * 512, "stages hold the sums of a tile");
  const cuuint64_t wd[3] = {(cuuint64_t)p.K, (cuuint64_t)p.N, (cuuint64_t)p.args.E * kHalves};
  const cuuint64_t wst[2] = {(cuuint64_t)p.K, (cuuint64_t)p.N * (cuuint64_t)p.K};
  const cuuint32_t wb[3] = {kBlk, kRowsW, 1};
  const cuuint64_t ad[2] = {(cuuint64_t)p.K, (cuuint64_t)p.M};
  const cuuint64_t ast[1] = {(cuuint64_t)p.lda};
  const cuuint32_t ab[2] = {kBlk, kTok};
  CUtensorMap tm_w, tm_a;
  if (int rc = encode_bytes_map(p.b, 3, wd, wst, wb, &tm_w, "B")) return rc;
  if (int rc = encode_bytes_map(p.a, 2, ad, ast, ab, &tm_a, "A")) return rc;
  const int64_t n_tiles = (p.N + kRowsW - 1) / kRowsW, groups = most_groups(p, kTok);
  if (groups > 65535 || n_tiles > 0x7fffffffLL / 8)
    return fail(MAGI_SWIGLU_ERR_SHAPE, "M=%lld rows are too many for one launch", (long long)p.M);
  Args args = p.args;
  args.splits = splits;
  args.stages = kStages;
  static int smem_set[kMaxDevices];
  cudaError_t e = allow_smem_once(fp8_block_stream_kernel<kHalves, kTok>, kSmem, device, smem_set);
  if (e != cudaSuccess) return fail_cuda(e, "cudaFuncSetAttribute(MaxDynamicSharedMemorySize)");
  e = launch(fp8_block_stream_kernel<kHalves, kTok>, dim3((unsigned)(n_tiles * args.splits), (unsigned)groups),
             dim3(kStreamThreads), kSmem, stream, (unsigned)args.splits, true, tm_w, tm_a, args);
  return e == cudaSuccess ? 0 : fail_cuda(e, "launch of fp8_block_stream_kernel");
}

// Clusters of 1, 2 and 4 CTA pairs that the GPU holds at once, per device and form (first entry 0: not queried yet).
static int g_tile_clusters[kMaxDevices][2][3];

template <int kHalves, int kCtas>
static int tile_ready() {
  cudaError_t e = cudaFuncSetAttribute(fp8_block_tile_kernel<kHalves, kCtas>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Tile<kCtas>::kSmem);
  if (e != cudaSuccess) return fail_cuda(e, "cudaFuncSetAttribute(MaxDynamicSharedMemorySize)");
  cudaFuncAttributes fa;
  e = cudaFuncGetAttributes(&fa, fp8_block_tile_kernel<kHalves, kCtas>);
  if (e != cudaSuccess) return fail_cuda(e, "cudaFuncGetAttributes");
  // the warpgroups' register shares add up to the launch's total: fewer at launch and the larger share would wait for good
  if (fa.numRegs != kTileRegs)
    return fail(MAGI_SWIGLU_ERR_DEVICE, "fp8_block_tile_kernel was built with %d registers a thread, not %d", fa.numRegs, kTileRegs);
  return 0;
}

template <int kHalves>
static int tile_clusters(int device, int sm_count, int (&clusters)[3]) {
  auto kernel = fp8_block_tile_kernel<kHalves, 2>;
  std::lock_guard<std::mutex> lock(g_dev_mutex);
  int(&known)[3] = g_tile_clusters[device][kHalves - 1];
  if (known[0] == 0) {
    if (int rc = tile_ready<kHalves, 1>()) return rc;
    if (int rc = tile_ready<kHalves, 2>()) return rc;
    cudaError_t e;
    int found[3] = {0, 0, 0};
    for (int i = 0; i < 3; ++i) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 2u << i;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.gridDim = dim3((unsigned)(sm_count / (2 << i) * (2 << i)));
      cfg.blockDim = dim3(kTileThreads);
      cfg.dynamicSmemBytes = Tile<2>::kSmem;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(&found[i], kernel, &cfg);
      if (e != cudaSuccess) return fail_cuda(e, "cudaOccupancyMaxActiveClusters");
    }
    if (found[0] < 1) return fail(MAGI_SWIGLU_ERR_DEVICE, "this device cannot hold a CTA pair of fp8_block_tile_kernel");
    for (int i = 0; i < 3; ++i) known[i] = found[i];
  }
  for (int i = 0; i < 3; ++i) clusters[i] = known[i];
  return 0;
}

// When all tiles fit as clusters of several pairs, those share the tiles' K blocks (at least eight each).
static int tile_log_splits(int64_t most, int kb, const int (&clusters)[3]) {
  int s = 0;
  while (s < 2 && most <= clusters[s + 1] && kb >= (16 << s)) ++s;
  return s;
}

template <int kHalves, int kCtas>
static int launch_tiles(const Problem& p, int splits, int most_workers, cudaStream_t stream) {
  constexpr int kTileRows = Tile<kCtas>::kRows;
  const cuuint64_t wd[3] = {(cuuint64_t)p.K, (cuuint64_t)p.N, (cuuint64_t)p.args.E * kHalves};
  const cuuint64_t wst[2] = {(cuuint64_t)p.K, (cuuint64_t)p.N * (cuuint64_t)p.K};
  const cuuint64_t ad[2] = {(cuuint64_t)p.K, (cuuint64_t)p.M};
  const cuuint64_t ast[1] = {(cuuint64_t)p.lda};
  const cuuint32_t wb[3] = {kBlk, 128, 1}, ab[2] = {kBlk, 128};
  CUtensorMap tm_w, tm_a;
  if (int rc = encode_bytes_map(p.b, 3, wd, wst, wb, &tm_w, "B")) return rc;
  if (int rc = encode_bytes_map(p.a, 2, ad, ast, ab, &tm_a, "A")) return rc;
  const int64_t n_tiles = (p.N + 256 / kHalves - 1) / (256 / kHalves);
  const int64_t units = most_groups(p, kTileRows);
  if (units * n_tiles > 0x7fffffffLL / 2) return fail(MAGI_SWIGLU_ERR_SHAPE, "M=%lld x N=%lld is too large for one launch", (long long)p.M, (long long)p.N);
  const int64_t most = units * n_tiles;
  Args args = p.args;
  args.splits = splits;
  // A raster band of about 32 MB of A: it is read once per column tile and should stay in L2 beside the W rows that pass
  // (8192 rows: K = 4096, N = 2 x 14336: bands of 8 / 16 / 32 groups 980 / 948 / 942 us; K = 14336: 447 / 451 / 468 us).
  const int64_t band = (32LL << 20) / (kTileRows * p.K);
  args.band = (int)(band < 4 ? 4 : (band > 64 ? 64 : band));
  const int64_t workers = most < most_workers ? most : most_workers;
  const int wide = ((uintptr_t)p.args.c & 31u) == 0 && p.N % 16 == 0;
  const cudaError_t e = launch(fp8_block_tile_kernel<kHalves, kCtas>, dim3((unsigned)(workers * kCtas * splits)),
                               dim3(kTileThreads), Tile<kCtas>::kSmem, stream, (unsigned)(kCtas * splits), false, tm_w, tm_a, args, wide);
  return e == cudaSuccess ? 0 : fail_cuda(e, "launch of fp8_block_tile_kernel");
}

// The kernel and its tokens per tile by what the forms are expected to take: rounds of the GPU's CTAs (pairs), each a
// fixed part and a part per K block.  The constants are microseconds measured with everything in flight (148 SMs):
// stream kernel, two CTAs an SM, 0.36 / 0.43 / 0.50 a K block for 16 / 32 / 64 tokens, 0.75 / 0.90 for 16 / 32 in the
// SwiGLU form, about 0.6 of that with one CTA an SM, and 3.0; tile kernel 0.42 a K block and 2.5 a tile.  Both sides at N = 4096,
// K = 14336 (stream 16 / 32 / 64 tokens, tiles): M = 64 26 / 18 / 16 / 35 us, 256 - / 47 / 35 / 35 us, 512 - / - / 58 /
// 37 us; SwiGLU, N = 1408, K = 2048, 64 experts (16 / 32 tokens, tiles): 512 rows 52 / 48 / 78 us, 2048 rows 85 / 75 / 96
// us, 8192 rows 295 / 199 / 138 us.  None is faster than W's bytes (6.2 TB/s).  Forms that are bound by them alike differ
// in what an uneven share costs: then the wider tile, up to 2.5 times the average share (8 experts, 74 rows, N = 4096, K =
// 14336: 16 tokens 69 to 87 us from routing to routing, 32 tokens 69 to 74 us).
static Form choose(const Problem& p, int sm_count, const int (&clusters)[3]) {
  const double n128 = (double)((p.N + 127) / 128);
  const double used = p.routed ? (double)(p.M < p.args.E ? p.M : p.args.E) : 1.0, share = p.M / used;
  const double bytes_us = used * p.halves * p.N * p.K / 6.2e6 + 3.0;
  double best = 0;
  int tok = 0, splits = 1;
  const int64_t n_tiles = (p.N * p.halves + 255) / 256;
  const int log_splits = tile_log_splits(most_groups(p, Tile<2>::kRows) * n_tiles, p.args.kb, clusters);
  // CTA pairs (256 rows) or single CTAs (128): half as much of a small expert's last group is padding, but a CTA fetches
  // 48 KB a K block and not 32, more yet when rows of K bytes start inside a 32-byte sector.  Pairs / singles, us: SwiGLU, 64
  // experts, 16040 rows, N = 1424: K = 1024 107 / 86, 2048 172 / 149, 4096 360 / 303, but 1040 117 / 123, 2064 191 / 217, 4112
  // 354 / 460; dense, 8192 rows, N = 4096: 1024 92 / 90, 2048 141 / 148, but 1040 101 / 130, 2064 161 / 226, 4112 293 / 437.  A
  // short K of this kind pays less than the rule expects (K = 528, the 64 experts: 87 / 78).  Other sizes: 64 experts, 6000
  // rows, N = 1408, K = 2048 128 / 91; 128 experts, 32768 rows, plain, N = 2048, K = 768 125 / 105; dense SwiGLU, N = 14336, K =
  // 4096: 384 rows 79 / 64, 8192 rows 1002 / 1052.  Both add in the same order.  Short K and few rows of many experts suit
  // single CTAs better than the stream kernel, whose CTAs are set up anew for every tile: plain, 128 experts, N = 2048, K = 768,
  // singles / 32 tokens: 1024 rows 35 / 48 us, 4096 rows 45 / 81.
  bool single = false;
  {
    const double rounds = rounds_of(p, expected_groups(p, Tile<2>::kRows) * n_tiles, clusters[log_splits]);
    best = 5.0 + rounds * (p.args.kb * 0.42 / (1 << log_splits) + 2.5) + (log_splits ? 3.0 : 0.0);
    const double rounds1 = rounds_of(p, expected_groups(p, Tile<1>::kRows) * n_tiles, sm_count);
    // warps without rows skip their work: nearly empty tiles take about 0.7 of a full one's time
    const double fill = share < 64 ? share / 64 : 1.0;
    const double cost1 = 3.0 + rounds1 * (p.args.kb * 0.42 + 2.5) * (p.K % 32 ? 1.5 : 1.12) * (0.7 + 0.3 * fill);
    if (cost1 < best) best = cost1, single = true;
    if (best < bytes_us) best = bytes_us;
  }
  const int forms = p.halves == 1 ? 3 : 2;
  static const double per_block[2][3] = {{0.36, 0.43, 0.50}, {0.75, 0.90, 0.0}};
  for (int i = 0; i < forms; ++i) {
    if (most_groups(p, 16 << i) > 65535) continue;
    const double ctas = n128 * expected_groups(p, 16 << i);
    int z = 1;  // up to eight CTAs of a cluster share a tile's K blocks, at least four each, until there are about two CTAs an SM
    while (z < 8 && ctas * z * 2 <= 2 * sm_count && p.args.kb >= z * 8) z *= 2;
    const double rounds = rounds_of(p, ctas * z, 2 * sm_count);
    double cost = 2.5 + rounds * (p.args.kb * per_block[p.halves - 1][i] / z * (ctas * z <= sm_count ? 0.6 : 1.0) + 3.0);
    if (cost < bytes_us) cost = bytes_us;
    if (cost < best || (cost == best && (tok == 0 || (p.routed && tok < 2.5 * share)))) best = cost, tok = 16 << i, splits = z;
  }
  if (tok) return Form{tok, 1, splits};
  return single ? Form{0, 1, 1} : Form{0, 2, 1 << log_splits};
}

// The form MAGI_SWIGLU_TUNE_FP8_FORM asks for, if it can serve this call.
static int forced(const Problem& p, int value, const int (&clusters)[3], Form* f) {
  const int base = value & 255, z = value >> 8;
  bool ok = false;
  if (base == 16 || base == 32 || (base == 64 && p.halves == 1)) {
    *f = Form{base, 1, z ? z : 1};
    ok = (z == 0 || z == 1 || z == 2 || z == 4 || z == 8) && f->splits <= p.args.kb && most_groups(p, base) <= 65535;
  } else if (base == 1 && z == 0) {
    *f = Form{0, 1, 1};
    ok = true;
  } else if ((base == 2 || base == 4 || base == 8) && z == 0) {
    *f = Form{0, 2, base / 2};
    const int64_t tiles = most_groups(p, Tile<2>::kRows) * ((p.N * p.halves + 255) / 256);
    ok = base == 2 || (f->splits <= p.args.kb && tiles <= clusters[base / 4]);
  }
  return ok ? 0 : fail(MAGI_SWIGLU_ERR_VARIANT, "form %d of the fp8 products cannot serve this call", value);
}

static int form_of(const Problem& p, int sm_count, const int (&clusters)[3], Form* f) {
  if (const int value = g_fp8_form.load(std::memory_order_relaxed)) return forced(p, value, clusters, f);
  *f = choose(p, sm_count, clusters);
  return 0;
}

static int run(const Problem& p, int device, void* cuda_stream) {
  const DeviceInfo* di = nullptr;
  if (int rc = require_b200(device, &di)) return rc;
  DeviceGuard guard;
  cudaError_t e = guard.set(device);
  if (e != cudaSuccess) return fail_cuda(e, "cudaSetDevice");
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  int clusters[3];
  if (int rc = p.halves == 1 ? tile_clusters<1>(device, di->sm_count, clusters) : tile_clusters<2>(device, di->sm_count, clusters))
    return rc;
  Form f;
  if (int rc = form_of(p, di->sm_count, clusters, &f)) return rc;
  const int pairs = f.tok ? 0 : clusters[f.splits >> 1];  // workers of 1, 2 or 4 pairs
  if (p.halves == 1) {
    if (f.tok == 16) return launch_stream<1, 16>(p, device, f.splits, stream);
    if (f.tok == 32) return launch_stream<1, 32>(p, device, f.splits, stream);
    if (f.tok == 64) return launch_stream<1, 64>(p, device, f.splits, stream);
    return f.ctas == 1 ? launch_tiles<1, 1>(p, 1, di->sm_count, stream) : launch_tiles<1, 2>(p, f.splits, pairs, stream);
  }
  if (f.tok == 16) return launch_stream<2, 16>(p, device, f.splits, stream);
  if (f.tok == 32) return launch_stream<2, 32>(p, device, f.splits, stream);
  return f.ctas == 1 ? launch_tiles<2, 1>(p, 1, di->sm_count, stream) : launch_tiles<2, 2>(p, f.splits, pairs, stream);
}

static int check(const void* a, const float* a_scale, const void* b, const float* b_scale, const int32_t* offsets,
                 int num_experts, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ld_scale, int n_multiple) {
  if (M < 0 || N < 1 || K < 1 || M > 0x3fffffffLL || N > 0x3fffffffLL || K > 0x3fffffffLL)
    return fail(MAGI_SWIGLU_ERR_SHAPE, "M=%lld, N=%lld, K=%lld out of range", (long long)M, (long long)N, (long long)K);
  if (N % n_multiple || K % 16)
    return fail(MAGI_SWIGLU_ERR_SHAPE, "N=%lld must be a multiple of %d and K=%lld of 16", (long long)N, n_multiple, (long long)K);
  if (num_experts < 1 || num_experts > 1024 || (!offsets && num_experts != 1))
    return fail(MAGI_SWIGLU_ERR_SHAPE, "num_experts=%d out of range [1, 1024], or more than one without offsets", num_experts);
  if (lda < K || ld_scale < (K + 127) / 128)
    return fail(MAGI_SWIGLU_ERR_SHAPE, "row strides too small: lda=%lld (K=%lld), ld_scale=%lld", (long long)lda, (long long)K, (long long)ld_scale);
  if (M == 0) return 0;
  if (!a || !a_scale || !b || !b_scale) return fail(MAGI_SWIGLU_ERR_NULL, "null pointer argument");
  if (lda % 16 || (((uintptr_t)a | (uintptr_t)b) & 15u))
    return fail(MAGI_SWIGLU_ERR_ALIGN, "a and b must be 16-byte aligned, and lda a multiple of 16");
  if ((((uintptr_t)a_scale | (uintptr_t)b_scale | (uintptr_t)offsets) & 3u))
    return fail(MAGI_SWIGLU_ERR_ALIGN, "scales and offsets must be 4-byte aligned");
  return 0;
}

static Problem problem(const void* a, const float* a_scale, const void* b, const float* b_scale, const int32_t* offsets,
                       int num_experts, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ld_scale, int zero_tail,
                       int halves) {
  Problem p;
  memset(&p, 0, sizeof(p));
  p.a = a;
  p.b = b;
  p.lda = lda;
  p.M = M;
  p.N = N;
  p.K = K;
  p.halves = halves;
  p.routed = offsets != nullptr;
  p.args.a_scale = a_scale;
  p.args.b_scale = b_scale;
  p.args.offsets = offsets;
  p.args.ld_as = ld_scale;
  p.args.R = (int)M;
  p.args.N = (int)N;
  p.args.E = num_experts;
  p.args.kb = (int)((K + kBlk - 1) / kBlk);
  p.args.nb = (int)((N + kBlk - 1) / kBlk);
  p.args.zero_tail = zero_tail;
  return p;
}

}  // namespace fp8
}  // namespace magi

using namespace magi;

extern "C" {

int magi_swiglu_gemm_fp8_block(const void* a, const float* a_scale, const void* b, const float* b_scale,
                               const int32_t* offsets, int num_experts, void* c, int64_t M, int64_t N, int64_t K,
                               int64_t lda, int64_t ld_scale, int zero_tail, int device, void* cuda_stream) {
  g_err[0] = 0;
  if (int rc = fp8::check(a, a_scale, b, b_scale, offsets, num_experts, M, N, K, lda, ld_scale, 8)) return rc;
  if (M == 0) return 0;
  if (!c) return fail(MAGI_SWIGLU_ERR_NULL, "null pointer argument");
  if ((uintptr_t)c & 15u) return fail(MAGI_SWIGLU_ERR_ALIGN, "c must be 16-byte aligned");
  fp8::Problem p = fp8::problem(a, a_scale, b, b_scale, offsets, num_experts, M, N, K, lda, ld_scale, zero_tail, 1);
  p.args.c = static_cast<__nv_bfloat16*>(c);
  return fp8::run(p, device, cuda_stream);
}

int magi_swiglu_gemm_swiglu_fp8_block(const void* a, const float* a_scale, const void* w_gate_up, const float* w_scale,
                                      const int32_t* offsets, int num_experts, void* codes, float* scales, int64_t M,
                                      int64_t N, int64_t K, int64_t lda, int64_t ld_scale, int zero_tail, int device,
                                      void* cuda_stream) {
  g_err[0] = 0;
  if (int rc = fp8::check(a, a_scale, w_gate_up, w_scale, offsets, num_experts, M, N, K, lda, ld_scale, 16)) return rc;
  if (M == 0) return 0;
  if (!codes || !scales) return fail(MAGI_SWIGLU_ERR_NULL, "null pointer argument");
  if (((uintptr_t)codes & 15u) || ((uintptr_t)scales & 3u))
    return fail(MAGI_SWIGLU_ERR_ALIGN, "codes must be 16-byte aligned and scales 4-byte aligned");
  fp8::Problem p = fp8::problem(a, a_scale, w_gate_up, w_scale, offsets, num_experts, M, N, K, lda, ld_scale, zero_tail, 2);
  p.args.codes = static_cast<uint8_t*>(codes);
  p.args.scales = scales;
  return fp8::run(p, device, cuda_stream);
}

int magi_swiglu_fp8_block_plan(int halves, int64_t M, int64_t N, int64_t K, int num_experts, int device, int sm_count,
                               int32_t out[4]) {
  g_err[0] = 0;
  if (!out) return fail(MAGI_SWIGLU_ERR_NULL, "out is null");
  if ((halves != 1 && halves != 2) || M < 1 || N < 1 || K < 1 || M > 0x3fffffffLL || N > 0x3fffffffLL || K > 0x3fffffffLL ||
      N % (8 * halves) || K % 16 || num_experts < 0 || num_experts > 1024)
    return fail(MAGI_SWIGLU_ERR_SHAPE, "halves=%d, M=%lld, N=%lld, K=%lld, num_experts=%d out of range", halves, (long long)M,
                (long long)N, (long long)K, num_experts);
  int clusters[3] = {sm_count / 2, sm_count / 4, sm_count / 8};
  if (sm_count <= 0) {
    const DeviceInfo* di = nullptr;
    if (int rc = require_b200(device, &di)) return rc;
    DeviceGuard guard;
    const cudaError_t e = guard.set(device);
    if (e != cudaSuccess) return fail_cuda(e, "cudaSetDevice");
    sm_count = di->sm_count;
    if (int rc = halves == 1 ? fp8::tile_clusters<1>(device, sm_count, clusters) : fp8::tile_clusters<2>(device, sm_count, clusters))
      return rc;
  }
  fp8::Problem p = fp8::problem(nullptr, nullptr, nullptr, nullptr, nullptr, num_experts ? num_experts : 1, M, N, K, K,
                                (K + 127) / 128, 0, halves);
  p.routed = num_experts > 0;
  fp8::Form f;
  if (int rc = fp8::form_of(p, sm_count, clusters, &f)) return rc;
  out[0] = f.tok, out[1] = f.ctas, out[2] = f.splits, out[3] = 0;
  return 0;
}

int magi_swiglu_fp8_block_watchdog_selftest(int device, void* cuda_stream, int64_t limit_cycles) {
  g_err[0] = 0;
  if (limit_cycles < 1000 || limit_cycles > 2000000000LL)
    return fail(MAGI_SWIGLU_ERR_SHAPE, "limit_cycles=%lld out of range [1000, 2e9]", (long long)limit_cycles);
  if (!device_info(device)) return fail(MAGI_SWIGLU_ERR_DEVICE, "device %d is not available", device);
  DeviceGuard guard;
  cudaError_t e = guard.set(device);
  if (e != cudaSuccess) return fail_cuda(e, "cudaSetDevice");
  fp8::fp8_watchdog_selftest_kernel<<<1, 32, 0, static_cast<cudaStream_t>(cuda_stream)>>>((long long)limit_cycles);
  e = cudaGetLastError();
  return e == cudaSuccess ? 0 : fail_cuda(e, "launch of fp8_watchdog_selftest_kernel");
}

}  // extern "C"
