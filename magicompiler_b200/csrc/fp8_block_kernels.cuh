// Device code of the block-scaled fp8 products:
//
//   C[m, n] = sum over K blocks b of  as[m, b] * bs[n / 128, b] * ( sum over k in block b of  a[m, k] * w[n, k] )
//
// with e4m3 codes, one fp32 scale per row and 128 K elements of A and one per 128 x 128 block of W; and the fused SwiGLU
// form, whose result silu(g) * u is quantised again in the same way (e4m3, one scale per row and 128 columns) without ever
// being written in a wider type.  With `offsets`, rows [offsets[e], offsets[e+1]) of A meet expert e's W.
//
// The inner sums run on the tensor cores (tcgen05 kind::f8f6f4, fp32 in tensor memory); the scales are not powers of two,
// so every K block of 128 is finished in tensor memory, read back, scaled and added to fp32 registers.  Several accumulator
// buffers in tensor memory (four in the stream kernel, two in the tile kernel) let the MMAs of the next blocks run meanwhile.
//
// fp8_block_stream_kernel: W's rows are the MMA's 128 rows ("M") and the tokens are its columns ("N", 16..64), so few
// tokens cost few MMA columns and few additions, and the kernel is a stream over W.  A CTA owns 128 output columns (128
// gate rows and 128 up rows of W in the SwiGLU form) of up to kTok rows of one expert.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "fp8_format.cuh"
#include "ptx_sm100.cuh"

namespace magi {
namespace fp8 {

constexpr int kBlk = 128;                 // K elements (= bytes) per scale block and pipeline stage: one swizzle row
constexpr int kRowsW = 128;               // rows of W per tile = tensor-memory lanes
constexpr int kWTile = kRowsW * kBlk;     // bytes
constexpr int kMaxStages = 8;
constexpr long long kWaitLimit = 6000000000LL;  // three to four seconds of SM cycles

__device__ unsigned int g_fp8_watchdog[4];  // {role that gave up, block, stage/buffer, parity}

// Bounded wait: after kWaitLimit the waiting role records itself, raises the CTA's abort flag and every role leaves.
__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity, volatile int* abort_flag, unsigned role,
                                             unsigned idx, long long limit = kWaitLimit) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  unsigned spins = 0;
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((++spins & 255u) == 0u) {
      if (*abort_flag) return false;
      if (clock64() - t0 > limit) {
        *abort_flag = 1;
        if (atomicCAS(&g_fp8_watchdog[0], 0u, role) == 0u) {
          g_fp8_watchdog[1] = blockIdx.x;
          g_fp8_watchdog[2] = idx;
          g_fp8_watchdog[3] = parity;
        }
        return false;
      }
    }
  }
}

// The same for a whole warp whose lanes wait for different barriers at the same time: a wait takes about a hundred cycles
// even when it is over, and waits one after the other add up on an MMA issuer's way.
__device__ __forceinline__ bool wait_bounded_all(uint32_t bar, uint32_t parity, volatile int* abort_flag, unsigned role,
                                                 unsigned idx) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity) != 0)) return true;
  const long long t0 = clock64();
  unsigned spins = 0;
  while (true) {
    const bool here = mbar_try_wait(bar, parity) != 0;
    if (__all_sync(0xffffffffu, here)) return true;
    if ((++spins & 255u) == 0u) {
      const bool late = clock64() - t0 > kWaitLimit;
      if (late && !here) {
        *abort_flag = 1;
        if (atomicCAS(&g_fp8_watchdog[0], 0u, role) == 0u) {
          g_fp8_watchdog[1] = blockIdx.x;
          g_fp8_watchdog[2] = idx;
          g_fp8_watchdog[3] = parity;
        }
      }
      if (__any_sync(0xffffffffu, late || *abort_flag != 0)) return false;
    }
  }
}

// The wait by itself, on a barrier that nothing signals: records {role 7, block 0, index 43, parity 0} after `limit` cycles.
__global__ void fp8_watchdog_selftest_kernel(long long limit) {
  __shared__ __align__(8) uint64_t bar;
  __shared__ int abort_flag;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    mbar_init(smem_u32(&bar), 1);
    fence_barrier_init();
  }
  __syncthreads();
  if (threadIdx.x == 0) wait_bounded(smem_u32(&bar), 0u, &abort_flag, 7u, 43u, limit);
  __syncthreads();
}

struct Args {
  const float* a_scale;   // [R, kb] fp32, row stride ld_as
  const float* b_scale;   // [E][halves * nb][kb]
  const int* offsets;     // [E + 1], or null: one expert with all R rows
  __nv_bfloat16* c;       // plain: [R, N]
  uint8_t* codes;         // SwiGLU: [R, N]
  float* scales;          // SwiGLU: [R, nb]
  long long ld_as;
  int R, N, E, kb, nb;    // nb = ceil(N / 128)
  int splits;             // CTAs (tile kernel: CTA pairs) of a cluster that share a tile's K blocks
  int stages;
  int zero_tail;          // rows from offsets[E] on: 1 = written as zeros, 0 = left alone
  int band;               // row groups a raster band of the tile kernel
  int never;              // 0; a condition that the compiler cannot fold
};

struct Unit {  // rows [row0, row0 + rows) of expert e; e == E: rows behind the last expert's; rows == 0: nothing
  int e, row0, rows;
};

__device__ __forceinline__ int warp_scan(int n) {  // inclusive sum over the warp's lanes
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, n, d);
    if (lane >= d) n += up;
  }
  return n;
}

// Rows [first, first + rows) of expert e, this lane's (the whole warp calls this, 32 experts at a time in order; `from`
// starts at 0); e == E: the rows behind the last expert's; beyond: none.  A bad array leads neither outside the operands nor
// to more groups than the host has counted on: offsets are clamped to [0, R], and one below an earlier one counts as that
// one, so that no row belongs to two experts.  Without offsets one expert has all rows.
struct Rows {
  int first, count;
};
__device__ __forceinline__ Rows rows_of(const Args& a, int e, int& from) {
  int lo = 0, next = 0;
  if (e <= a.E) {
    lo = a.offsets ? min(max(a.offsets[e], 0), a.R) : (e == 0 ? 0 : a.R);
    next = a.offsets && e < a.E ? min(max(a.offsets[e + 1], 0), a.R) : a.R;
  }
  if (__any_sync(0xffffffffu, e <= a.E && (lo < from || next < lo))) {  // never for offsets as they should be
    lo = max(lo, from);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) lo = max(lo, __shfl_up_sync(0xffffffffu, lo, d));  // a lane below d gets its own
  }
  from = __shfl_sync(0xffffffffu, lo, 31);
  return Rows{lo, e <= a.E ? max(next - lo, 0) : 0};
}

// The unit-th group of at most kTok rows, counting every expert's groups in order (one whole warp calls this).
template <int kTok>
__device__ __forceinline__ Unit find_unit(const Args& a, int unit) {
  const int lane = threadIdx.x & 31;
  int seen = 0, from = 0;
  for (int b = 0; b <= a.E; b += 32) {
    const int e = b + lane;
    const Rows r = rows_of(a, e, from);
    const int n = (e == a.E && !a.zero_tail) ? 0 : (r.count + kTok - 1) / kTok;
    const int scan = warp_scan(n);
    const unsigned hit = __ballot_sync(0xffffffffu, n > 0 && unit >= seen + scan - n && unit < seen + scan);
    if (hit) {
      const int src = __ffs(hit) - 1, i = unit - seen - __shfl_sync(0xffffffffu, scan - n, src);
      const int first = __shfl_sync(0xffffffffu, r.first, src), rows = __shfl_sync(0xffffffffu, r.count, src);
      return Unit{b + src, first + i * kTok, min(kTok, rows - i * kTok)};
    }
    seen += __shfl_sync(0xffffffffu, scan, 31);
  }
  return Unit{0, 0, 0};
}

__device__ __forceinline__ float silu_mul(float g, float u) {
  return g * rcp_approx(1.0f + ex2_approx(-1.4426950408889634f * g)) * u;
}
__device__ __forceinline__ float warp_max_nan(float v) {  // maximum of non-negative values and NaN, NaN wins
  unsigned b = __float_as_uint(v);
#pragma unroll
  for (int o = 16; o; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
  return __uint_as_float(b);
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_shared_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_v4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
__device__ __forceinline__ void st_shared_f32(uint32_t addr, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void epilogue_sync(int threads) {  // named barrier of the epilogue warps
  asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
}

constexpr int kStreamThreads = 192;  // warps 0-3 epilogue (one tensor-memory lane quarter each), 4 TMA producer, 5 MMA issuer

// kTok 16, 32 or (plain) 64 tokens a tile: two CTAs share an SM.  (Tiles of 64 tokens in the SwiGLU form and of 128 in the
// plain one leave registers for one CTA an SM only and lost to the smaller ones everywhere.)  kBufs accumulator buffers: a
// buffer's way from the MMA through the epilogue and back takes about 700 cycles besides the MMA itself, which takes 400.
// Blocks set up (barriers, tensor memory, descriptors) while the previous kernel drains: 75.8 to 72.7 us back to back for 16
// tokens, K 8192, N 28672; a routed fp8 block in a graph 68.7 to 66.4 us (1 token, 2 of 8 experts, K 4096, N 14336), 25.0
// to 24.2 (8 of 128, K 2048, N 768), but 205 to 209 for 64 tokens, 8 of 256 experts.
template <int kHalves, int kTok>
__global__ void __launch_bounds__(kStreamThreads, 2)
fp8_block_stream_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a, const Args a) {
  constexpr int kATile = kTok * kBlk;
  constexpr int kStage = kHalves * kWTile + kATile;
  constexpr int kAccCols = kHalves * kTok;
  constexpr int kBufs = 4;
  constexpr int kTmem = kBufs * kAccCols;
  constexpr int kPiece = kAccCols < 32 ? kAccCols : 32;  // columns per tensor-memory load
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(16) float ring[2][4][kAccCols];  // as * bs of four K blocks: every column of both halves
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 2 * kBufs];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ Unit unit_slot;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (kMaxStages + s); };
  auto acc_full = [&](int b) { return bar0 + 8u * (2 * kMaxStages + b); };
  auto acc_empty = [&](int b) { return bar0 + 8u * (2 * kMaxStages + kBufs + b); };
  const int split = a.splits > 1 ? (int)cluster_ctarank() : 0;
  const int n0 = (int)(blockIdx.x / a.splits) * kRowsW;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < kBufs; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), 4);
    }
    fence_barrier_init();
  }
  if (warp == 5) {
    tmem_alloc<1>(smem_u32(&tmem_slot), kTmem);
    tmem_relinquish<1>();
  }
  if (warp == 4) {
    grid_dependency_wait();
    const Unit found = find_unit<kTok>(a, blockIdx.y);
    if (lane == 0) unit_slot = found;
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  grid_launch_dependents();  // after the allocation: a later kernel cannot take the tensor memory this one still needs
  grid_dependency_wait();
  const uint32_t tmem = tmem_slot;
  const Unit u = unit_slot;
  const bool live = u.rows > 0 && u.e < a.E;  // the same for every CTA of a cluster
  const int kb0 = (int)((long long)a.kb * split / a.splits), kb1 = (int)((long long)a.kb * (split + 1) / a.splits);

  if (live && warp == 4 && lane == 0) {
    // ------------------------------------------------------------ TMA producer
    prefetch_tensormap(&tm_w);
    prefetch_tensormap(&tm_a);
    const uint64_t keep = l2_policy_evict_last(), once = l2_policy_evict_first();
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!wait_bounded(empty_bar(stage), phase ^ 1u, &abort_flag, 1u, stage)) break;
      mbar_arrive_expect_tx(full_bar(stage), kStage);
      const uint32_t dst = tiles + stage * kStage;
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
        tma_load_3d_hint(dst + h * kWTile, &tm_w, full_bar(stage), kb * kBlk, n0, u.e * kHalves + h, once);
      tma_load_2d_hint(dst + kHalves * kWTile, &tm_a, full_bar(stage), kb * kBlk, u.row0, keep);
      if (++stage == a.stages) stage = 0, phase ^= 1u;
    }
  } else if (live && warp == 5) {
    // ------------------------------------------------------------ MMA issuer
    const uint32_t idesc = umma_idesc_e4m3(kRowsW, kTok);
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int buf = (kb - kb0) % kBufs;
      if (!wait_bounded_all(lane == 0 ? full_bar(stage) : acc_empty(buf), lane == 0 ? phase : (((kb - kb0) / kBufs) & 1) ^ 1u,
                            &abort_flag, 2u, lane == 0 ? stage : 16 + buf))
        break;
      tc_fence_after_sync();
      if (lane == 0) {
        const uint32_t src = tiles + stage * kStage;
        const uint64_t tok = umma_desc_k_sw128(src + kHalves * kWTile);
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          const uint64_t w = umma_desc_k_sw128(src + h * kWTile);
#pragma unroll
          for (int i = 0; i < kBlk / 32; ++i)
            umma_fp8<1>(tmem + buf * kAccCols + h * kTok, w + 2 * i, tok + 2 * i, idesc, i > 0);
        }
        umma_commit<1>(acc_full(buf));
        umma_commit<1>(empty_bar(stage));
      }
      __syncwarp();
      if (++stage == a.stages) stage = 0, phase ^= 1u;
    }
  } else if (live && warp < 4) {
    // ------------------------------------------------------------ scale and add (one row of W per thread)
    uint64_t sum[kAccCols / 2];  // pairs of neighbouring columns
#pragma unroll
    for (int c = 0; c < kAccCols / 2; ++c) sum[c] = 0;
    // Scales travel four K blocks at a time: a prefetch into registers, then their products into half of a shared ring.
    constexpr int kLoads = (4 * kTok + 127) / 128;
    float next[kLoads], next_w[kHalves];
    const float* ws = a.b_scale + ((long long)u.e * kHalves * a.nb + n0 / kBlk) * a.kb;
    auto fetch = [&](int kb) {  // thread i holds token i / 4 (and every 32nd after it) at K block kb + i % 4
      const int b = kb + (threadIdx.x & 3);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int c = (threadIdx.x >> 2) + 32 * i;
        next[i] = (c < u.rows && c < kTok && b < kb1) ? a.a_scale[(long long)(u.row0 + c) * a.ld_as + b] : 0.0f;
      }
#pragma unroll
      for (int h = 0; h < kHalves; ++h) next_w[h] = b < kb1 ? ws[(long long)h * a.nb * a.kb + b] : 0.0f;
    };
    fetch(kb0);
    const uint32_t lane_base = tmem + ((uint32_t)(warp * 32) << 16);
    bool ok = true;
    int never = a.never;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int i = kb - kb0, half = (i >> 2) & 1, buf = i % kBufs;
      if ((i & 3) == 0) {
        // everyone is past the previous four blocks, so the other half of the ring is free
#pragma unroll
        for (int q = 0; q < kLoads; ++q) {
          const int c = (threadIdx.x >> 2) + 32 * q;
          if (c < kTok)
#pragma unroll
            for (int h = 0; h < kHalves; ++h) ring[half][threadIdx.x & 3][h * kTok + c] = next[q] * next_w[h];
        }
        epilogue_sync(128);
        fetch(kb + 4);
      }
      // a wait that gave up skips the work but not the barrier above, which the other warps are counting on
      ok = __all_sync(0xffffffffu, ok && wait_bounded(acc_full(buf), (i / kBufs) & 1, &abort_flag, 3u, buf));
      if (!ok) continue;
      tc_fence_after_sync();
      const uint32_t sc = smem_u32(ring[half][i & 3]);
      uint32_t p[kAccCols / kPiece][32];
#pragma unroll
      for (int j = 0; j < kAccCols / kPiece; ++j) {
        if constexpr (kPiece == 32)
          tmem_ld_x32(lane_base + buf * kAccCols + 32 * j, p[j]);
        else
          tmem_ld_x16_into32(lane_base + buf * kAccCols, p[j]);
      }
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < kAccCols / kPiece; ++j) tmem_regs_ready(p[j]);
      tc_fence_before_sync();  // all columns have been read: the buffer goes back before the arithmetic
      __syncwarp();
      if (lane == 0) mbar_arrive_relaxed(acc_empty(buf));
      asm volatile("" : "+r"(never));  // see the tile kernel
      if (never) break;
#pragma unroll
      for (int c = 0; c < kAccCols; c += 4) {
        const uint32_t* v = p[c / kPiece] + c % kPiece;
        const float4 t = ld_shared_f4(sc + c * 4);
        fma_f32x2(sum[c / 2], v[0], v[1], pack_f32x2(t.x, t.y));
        fma_f32x2(sum[c / 2 + 1], v[2], v[3], pack_f32x2(t.z, t.w));
      }
    }
    float acc[kHalves][kTok];
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
      for (int c = 0; c < kTok; c += 2) unpack_f32x2(sum[(h * kTok + c) / 2], acc[h][c], acc[h][c + 1]);
    // Every MMA of this CTA is complete, so the stages are free: the sums go there as [token][half][128], which is
    // conflict-free here and gives the writer below a token's 128 columns in a row.
    const uint32_t mine = tiles + (warp * 32 + lane) * 4;
#pragma unroll
    for (int c = 0; c < kTok; ++c)
#pragma unroll
      for (int h = 0; h < kHalves; ++h) st_shared_f32(mine + (c * kHalves + h) * 512, acc[h][c]);
  }
  __syncwarp();
  if (live) {
    if (a.splits > 1)
      cluster_sync_all();
    else
      __syncthreads();
  }

  // ------------------------------------------------------------ output: one warp per token, four columns per lane
  if (warp < 4 && u.rows > 0) {
    const int n = n0 + 4 * lane;
    for (int c = split + a.splits * warp; c < u.rows; c += a.splits * 4) {
      float4 v[kHalves];
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        v[h] = make_float4(0, 0, 0, 0);
        if (!live) continue;
        const uint32_t at = tiles + (c * kHalves + h) * 512 + lane * 16;
        if (a.splits == 1) {
          v[h] = ld_shared_f4(at);
        } else {
          for (int z = 0; z < a.splits; ++z) {  // in split order: the same sum every time
            const float4 q = ld_cluster_f4(map_to_cta(at, z));
            v[h].x += q.x, v[h].y += q.y, v[h].z += q.z, v[h].w += q.w;
          }
        }
      }
      const long long row = u.row0 + c;
      if constexpr (kHalves == 1) {
        if (n < a.N) {
          const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0].x, v[0].y), hi = __floats2bfloat162_rn(v[0].z, v[0].w);
          uint2 o;
          o.x = *reinterpret_cast<const uint32_t*>(&lo);
          o.y = *reinterpret_cast<const uint32_t*>(&hi);
          *reinterpret_cast<uint2*>(a.c + row * a.N + n) = o;
        }
      } else {
        // columns beyond N hold zeros (W's rows there are zero-filled), which no maximum notices
        float y0 = silu_mul(v[0].x, v[1].x), y1 = silu_mul(v[0].y, v[1].y), y2 = silu_mul(v[0].z, v[1].z),
              y3 = silu_mul(v[0].w, v[1].w);
        unsigned top = max(max(__float_as_uint(fabsf(y0)), __float_as_uint(fabsf(y1))),
                           max(__float_as_uint(fabsf(y2)), __float_as_uint(fabsf(y3))));
        const float s = block_scale(warp_max_nan(__uint_as_float(top))), lift = lift_of(s);
        y0 *= lift, y1 *= lift, y2 *= lift, y3 *= lift;
        const Divisor d(s * lift);
        d.divide(y0, y1);
        d.divide(y2, y3);
        if (n < a.N) *reinterpret_cast<uint32_t*>(a.codes + row * a.N + n) = pack4_e4m3(y0, y1, y2, y3);
        if (lane == 0) a.scales[row * a.nb + n0 / kBlk] = s;
      }
    }
  }

  // ------------------------------------------------------------ teardown (also the abort path)
  __syncwarp();
  if (*reinterpret_cast<volatile int*>(&abort_flag)) {
    const long long t0 = clock64();  // copies and MMAs in flight land before tensor memory is freed
    while (clock64() - t0 < 4000000LL) {
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (live && a.splits > 1) cluster_sync_all();  // nobody leaves while its sums may still be read
  if (warp == 5) tmem_dealloc<1>(tmem, kTmem);
}

// ---------------------------------------------------------------- many rows an expert: CTA pairs
// fp8_block_tile_kernel: tokens are the MMA's rows.  A pair (tcgen05 cta_group::2) owns 256 rows of one expert and 256
// rows of W (256 output columns, or 128 gate and the matching 128 up columns); each CTA loads its own 128 rows of A and
// half of W's, 32 KB per K block for 512 cycles of MMA.  A thread of the epilogue owns one row, so its scale is one number
// per 128 columns and an addition is one fused multiply-add; with 128 of them per thread and block, two epilogue warps a
// scheduler keep up with the MMA (half of the issue slots) and the registers for them come from the other warpgroup.
// It is launched without programmatic overlap (the extra wait changes the loop's instruction schedule for the worse).
// Persistent: tiles go round-robin to the pairs in bands of row groups, column tile by column tile, so that the
// pairs that run together share A rows and W rows in L2.
// kCtas 1: the same loop for one CTA with 128 rows of A and all 256 of W, 48 KB a K block; less padding for small experts
// (SwiGLU, 64 experts, 6000 rows, N 1408, K 2048: 91 us against 128 with pairs), more L2 traffic (8192 dense rows, N 14336,
// K 4096: 1052 against 1002).  Additions come in the same order: the results are the same bits.
// Few tiles: `splits` (2 or 4) pairs form a cluster and share a tile's K blocks.  At the end each pair keeps the rows of
// 4 / splits lane quarters, sends the sums of the others to the pairs that keep those (distributed shared memory, into the
// stages, which are free by then) and adds what it receives in the order of the splits.  One tile a cluster: the host splits
// only what fits, and rows_of makes no more groups than the host counts on, whatever the offsets hold.
constexpr int kTileThreads = 384;  // warps 0 TMA, 1 and 3 MMA, 2 tensor-memory allocator and scales; 4-11 epilogue
constexpr int kTileRegs = 168;     // a thread's registers at launch: 384 * 168 = 64512 = 128 * 56 + 256 * 224
template <int kCtas>
struct Tile {
  static constexpr int kRows = 128 * kCtas;
  static constexpr int kStage = kCtas == 2 ? 2 * kWTile : 3 * kWTile;
  static constexpr int kStages = kCtas == 2 ? 6 : 4;
  static constexpr int kSmem = kStages * kStage + 1024;
};
constexpr int kMapExperts = 1024;
constexpr int kScaleSlots = 4;     // ring of scale products, four K blocks a slot

struct TileAt {
  int e, row0, end, n0;  // rows [row0, min(row0 + kRows, end)), first output column
};
constexpr int kTileInfos = 2 * kScaleSlots;  // the scale warp is at most kScaleSlots tiles ahead

template <int kHalves, int kCtas>
__global__ void __launch_bounds__(kTileThreads, 1)
fp8_block_tile_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a, const Args a,
                      const int wide_store) {
  constexpr int kOutCols = 256 / kHalves;
  constexpr int kTileRows = Tile<kCtas>::kRows, kTileStage = Tile<kCtas>::kStage, kTileStages = Tile<kCtas>::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int row_start[kMapExperts + 1], unit_first[kMapExperts + 1];
  __shared__ unsigned top_half[2][128];
  __shared__ TileAt tile_info[kTileInfos];
  __shared__ float scale_ring[kScaleSlots][4][2][128];  // as * bs of each row with both 128-column blocks of the tile
  __shared__ __align__(8) uint64_t bars[2 * kTileStages + 4 + 2 * kScaleSlots];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cluster_rank = (int)cluster_ctarank();
  const int rank = kCtas == 2 ? cluster_rank & 1 : 0, split = kCtas == 2 ? cluster_rank >> 1 : 0;  // rank 0 issues the pair's MMAs
  const uint32_t leader = kCtas == 2 ? cluster_rank & ~1 : 0;
  const uint16_t both = (uint16_t)(3u << leader);
  const int pair = blockIdx.x / (kCtas * a.splits), pairs = gridDim.x / (kCtas * a.splits);  // pairs, or clusters of them
  const int kb0 = (int)((long long)a.kb * split / a.splits), kb1 = (int)((long long)a.kb * (split + 1) / a.splits);
  const uint32_t tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (kTileStages + s); };
  auto acc_full = [&](int b) { return bar0 + 8u * (2 * kTileStages + b); };
  auto acc_empty = [&](int b) { return bar0 + 8u * (2 * kTileStages + 2 + b); };
  auto scale_full = [&](int s) { return bar0 + 8u * (2 * kTileStages + 4 + s); };
  auto scale_empty = [&](int s) { return bar0 + 8u * (2 * kTileStages + 4 + kScaleSlots + s); };

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kTileStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), 8 * kCtas);  // the epilogue warps of both CTAs
    }
    for (int s = 0; s < kScaleSlots; ++s) {
      mbar_init(scale_full(s), 1);
      mbar_init(scale_empty(s), 8);
    }
    fence_barrier_init();
    prefetch_tensormap(&tm_w);
    prefetch_tensormap(&tm_a);
  }
  if (warp == 2) {
    tmem_alloc<kCtas>(smem_u32(&tmem_slot), 512);
    tmem_relinquish<kCtas>();
  }
  if (warp == 3) {  // where each expert's rows and row groups begin
    int seen = 0, from = 0;
    for (int b = 0; b <= a.E; b += 32) {
      const int e = b + lane;
      const Rows r = rows_of(a, e, from);
      const int n = e < a.E ? (r.count + kTileRows - 1) / kTileRows : 0, scan = warp_scan(n);
      if (e <= a.E) {
        row_start[e] = r.first;
        unit_first[e] = seen + scan - n;
      }
      seen += __shfl_sync(0xffffffffu, scan, 31);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers exist before anything signals them
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  const int n_tiles = (a.N + kOutCols - 1) / kOutCols;
  const int units = unit_first[a.E], total = units * n_tiles;

  auto locate = [&](int t) {
    TileAt at;
    const int band = t / (a.band * n_tiles), rem = t - band * a.band * n_tiles;
    const int high = min(a.band, units - band * a.band);
    const int unit = band * a.band + rem % high;
    at.n0 = rem / high * kOutCols;
    int lo = 0, hi = a.E;  // unit_first[lo] <= unit < unit_first[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (unit_first[mid] <= unit) lo = mid; else hi = mid;
    }
    at.e = lo;
    at.row0 = row_start[lo] + (unit - unit_first[lo]) * kTileRows;
    at.end = row_start[lo + 1];
    return at;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------- TMA producer (each CTA its own halves)
      const uint64_t keep = l2_policy_evict_last(), normal = l2_policy_evict_normal();
      const uint32_t full0 = map_to_cta(full_bar(0), leader);  // the bytes of both CTAs are counted on rank 0's barrier
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair; t < total && ok; t += pairs) {
        const TileAt at = locate(t);
        const int row = at.row0 + 128 * rank;
        // a CTA whose rows all lie behind the expert's end brings no A rows; what the MMA reads instead is never used
        const bool empty = row >= at.end, peer_empty = at.row0 + 128 >= at.end;
        const int wrow = kHalves == 1 ? at.n0 + 128 * rank : at.n0, whalf = kHalves == 1 ? at.e : at.e * 2 + rank;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = wait_bounded(empty_bar(stage), phase ^ 1u, &abort_flag, 1u, stage))) break;
          const uint32_t dst = tiles + stage * kTileStage;
          if constexpr (kCtas == 2) {
            if (rank == 0) mbar_arrive_expect_tx(full_bar(stage), 2 * kTileStage - (peer_empty ? kWTile : 0));
            if (!empty) tma_load_2d_pair_hint(dst, &tm_a, full0 + 8u * stage, kb * kBlk, row, keep);
            tma_load_3d_pair_hint(dst + kWTile, &tm_w, full0 + 8u * stage, kb * kBlk, wrow, whalf, normal);
          } else {
            mbar_arrive_expect_tx(full_bar(stage), kTileStage);
            tma_load_2d_hint(dst, &tm_a, full_bar(stage), kb * kBlk, row, keep);
            tma_load_3d_hint(dst + kWTile, &tm_w, full_bar(stage), kb * kBlk, wrow, whalf, normal);
            tma_load_3d_hint(dst + 2 * kWTile, &tm_w, full_bar(stage), kb * kBlk, kHalves == 1 ? wrow + 128 : wrow,
                             kHalves == 1 ? whalf : whalf + 1, normal);
          }
          if (++stage == kTileStages) stage = 0, phase ^= 1u;
        }
      }
    } else if ((warp == 1 || warp == 3) && rank == 0) {
      // ---------------------------------------------------------- MMA issuers: warp 1 the even K blocks, warp 3 the odd
      // ones, each with a buffer of its own.  Issuing four MMAs holds a thread until the tensor pipe has taken them, so two
      // issuers do their waits in each other's shadow; lane 0 waits for the operands while the others wait for the buffer.
      const uint32_t idesc = umma_idesc_e4m3(128 * kCtas, 256);
      const int buf = warp >> 1;
      int it = 0, stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair; t < total && ok; t += pairs)
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          if ((it & 1) == buf) {
            ok = wait_bounded_all(lane == 0 ? full_bar(stage) : acc_empty(buf), lane == 0 ? phase : ((it >> 1) & 1) ^ 1u,
                                  &abort_flag, 2u, lane == 0 ? stage : 16 + buf);
            if (!ok) break;
            tc_fence_after_sync();
            if (lane == 0) {
              const uint64_t da = umma_desc_k_sw128(tiles + stage * kTileStage);
              const uint64_t dw = umma_desc_k_sw128(tiles + stage * kTileStage + kWTile);
#pragma unroll
              for (int i = 0; i < kBlk / 32; ++i) umma_fp8<kCtas>(tmem + buf * 256, da + 2 * i, dw + 2 * i, idesc, i > 0);
              umma_commit<kCtas>(acc_full(buf), both);
              umma_commit<kCtas>(empty_bar(stage), both);
            }
            __syncwarp();
          }
          if (++stage == kTileStages) stage = 0, phase ^= 1u;
        }
    } else if (warp == 2) {
      // ---------------------------------------------------------- scales: the epilogue has no registers to spare for them
      int slot = 0, nth = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair; t < total && ok; t += pairs, ++nth) {
        const TileAt at = locate(t);
        const float* w0 = a.b_scale + ((long long)at.e * kHalves * a.nb + at.n0 / kBlk) * a.kb;
        // the tile's second block: the next 128 columns (none: any valid one), or the up half's
        const float* w1 = w0 + (kHalves == 2 ? (long long)a.nb * a.kb : (at.n0 / kBlk + 1 < a.nb ? a.kb : 0));
        const float* rows[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          rows[i] = a.a_scale + (long long)min(at.row0 + 128 * rank + 32 * i + lane, at.end - 1) * a.ld_as;
        for (int kb = kb0; kb < kb1; kb += 4) {
          if (!(ok = __all_sync(0xffffffffu, wait_bounded(scale_empty(slot), phase ^ 1u, &abort_flag, 4u, slot)))) break;
#pragma unroll
          for (int b = 0; b < 4; b += 2) {
            const int k0 = min(kb + b, kb1 - 1), k1 = min(kb + b + 1, kb1 - 1);
            float r0[4], r1[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) r0[i] = __ldg(rows[i] + k0), r1[i] = __ldg(rows[i] + k1);
            const float g0 = __ldg(w0 + k0), g1 = __ldg(w0 + k1), u0 = __ldg(w1 + k0), u1 = __ldg(w1 + k1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              scale_ring[slot][b][0][32 * i + lane] = r0[i] * g0;
              scale_ring[slot][b][1][32 * i + lane] = r0[i] * u0;
              scale_ring[slot][b + 1][0][32 * i + lane] = r1[i] * g1;
              scale_ring[slot][b + 1][1][32 * i + lane] = r1[i] * u1;
            }
          }
          __syncwarp();
          if (lane == 0) {
            if (kb == kb0) tile_info[nth % kTileInfos] = at;
            mbar_arrive(scale_full(slot));
          }
          if (++slot == kScaleSlots) slot = 0, phase ^= 1u;
        }
      }
    }
    __syncwarp();
    if (a.splits > 1 && pair < total) {  // the two barriers of the epilogue's exchange
      cluster_sync_all();
      cluster_sync_all();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    // ------------------------------------------------------------ scale, add, write: one row per thread
    const int q = warp & 3, part = (warp - 4) >> 2;  // lane quarter; which half of the columns
    const int my_row = 128 * rank + 32 * q + lane;
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
    const uint32_t acc_empty0 = map_to_cta(acc_empty(0), leader);
    // plain: 128 columns of one block of W; SwiGLU: 64 gate columns, then the 64 up columns that meet them
    const int col[4] = {kHalves == 1 ? 128 * part : 64 * part, kHalves == 1 ? 128 * part + 32 : 64 * part + 32,
                        kHalves == 1 ? 128 * part + 64 : 128 + 64 * part, kHalves == 1 ? 128 * part + 96 : 160 + 64 * part};
    const uint64_t c_policy = l2_policy_evict_first();
    int it = 0, slot = 0, never = a.never, nth = 0;
    uint32_t slot_phase = 0;
    bool ok = true;
    for (int t = pair; t < total; t += pairs, ++nth) {
      uint64_t sum[64];  // pairs of neighbouring columns
#pragma unroll
      for (int i = 0; i < 64; ++i) sum[i] = 0;
      for (int kb = kb0; kb < kb1; kb += 4) {
        ok = __all_sync(0xffffffffu, ok && wait_bounded(scale_full(slot), slot_phase, &abort_flag, 3u, 32 + slot));
        // a warp without rows only keeps the barriers going
        const bool idle = tile_info[nth % kTileInfos].row0 + 128 * rank + 32 * q >= tile_info[nth % kTileInfos].end;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (kb + i >= kb1) break;
          const float f0 = scale_ring[slot][i][kHalves == 1 ? part : 0][32 * q + lane];
          const float f1 = kHalves == 1 ? f0 : scale_ring[slot][i][1][32 * q + lane];
          const int buf = it & 1;
          ok = __all_sync(0xffffffffu, ok && wait_bounded(acc_full(buf), (it >> 1) & 1, &abort_flag, 3u, buf));
          ++it;
          if (!ok) continue;
          if (idle) {
            if (lane == 0) mbar_arrive_cluster_relaxed(acc_empty0 + 8u * buf);
            continue;
          }
          tc_fence_after_sync();
          const uint64_t s0 = pack_f32x2(f0, f0), s1 = pack_f32x2(f1, f1);
          const uint32_t from = lanes + buf * 256;
          // The buffer goes back as soon as the last columns have been read: everything before that is on the MMA's
          // critical path, so two loads are in flight and the arithmetic that can wait comes after the arrival.
          uint32_t p[32], q2[32];
          tmem_ld_x32(from + col[0], p);
          tmem_ld_x32(from + col[1], q2);
          tmem_ld_wait();
          tmem_regs_ready(p);
          tmem_regs_ready(q2);
#pragma unroll
          for (int j = 0; j < 16; ++j) fma_f32x2(sum[j], p[2 * j], p[2 * j + 1], s0);
          tmem_ld_x32(from + col[2], p);
#pragma unroll
          for (int j = 0; j < 16; ++j) fma_f32x2(sum[16 + j], q2[2 * j], q2[2 * j + 1], s0);
          tmem_ld_x32(from + col[3], q2);
          tmem_ld_wait();
          tmem_regs_ready(p);
          tmem_regs_ready(q2);
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(acc_empty0 + 8u * buf);
          // A branch that is never taken: instructions do not move across it, and without it the assembler puts the
          // arithmetic below in front of the arrival (1039 instead of 813 cycles a K block, K = 14336).
          asm volatile("" : "+r"(never));
          if (never) break;
#pragma unroll
          for (int j = 0; j < 16; ++j) fma_f32x2(sum[32 + j], p[2 * j], p[2 * j + 1], s1);
#pragma unroll
          for (int j = 0; j < 16; ++j) fma_f32x2(sum[48 + j], q2[2 * j], q2[2 * j + 1], s1);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(scale_empty(slot));
        if (++slot == kScaleSlots) slot = 0, slot_phase ^= 1u;
      }
      const TileAt at = tile_info[nth % kTileInfos];
      float acc[128];
#pragma unroll
      for (int i = 0; i < 64; ++i) unpack_f32x2(sum[i], acc[2 * i], acc[2 * i + 1]);
      bool keeps = true;
      if (a.splits > 1) {
        const int per = 4 / a.splits, keeper = q / per;  // lane quarters a pair keeps; which pair keeps this one
        keeps = split == keeper;
        // [sender][warp of the keeper][32 x 16 bytes][lane]
        const uint32_t slab = (uint32_t)((q % per) * 2 + part) * 16384u + lane * 16u;
        cluster_sync_all();  // every MMA of the cluster is complete: the stages are free
        if (!keeps) {
          const uint32_t sender = (uint32_t)(split < keeper ? split : split - 1) * (uint32_t)(per * 2) * 16384u;
          const uint32_t dst = map_to_cta(tiles + sender + slab, 2 * keeper + rank);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            st_cluster_v4(dst + i * 512, acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
        }
        cluster_sync_all();
        if (keeps)
          for (int s = 0; s < a.splits - 1; ++s) {
            const uint32_t src = tiles + (uint32_t)s * (uint32_t)(per * 2) * 16384u + slab;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float4 v = ld_shared_f4(src + i * 512);
              acc[4 * i] += v.x, acc[4 * i + 1] += v.y, acc[4 * i + 2] += v.z, acc[4 * i + 3] += v.w;
            }
          }
      }
      const long long row = at.row0 + my_row;
      const bool here = ok && keeps && row < at.end;
      if constexpr (kHalves == 1) {
        const int n = at.n0 + 128 * part;
        __nv_bfloat16* dst = a.c + row * a.N + n;
        if (here) {
#pragma unroll
          for (int j = 0; j < 128; j += 16) {
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const __nv_bfloat162 h = __floats2bfloat162_rn(acc[j + 2 * i], acc[j + 2 * i + 1]);
              o[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
            const uint4 lo = make_uint4(o[0], o[1], o[2], o[3]), hi = make_uint4(o[4], o[5], o[6], o[7]);
            if (wide_store) {  // 32-byte rows: N is a multiple of 16
              if (n + j < a.N) st_global_v8_hint(dst + j, lo, hi, c_policy);
            } else {
              if (n + j < a.N) *reinterpret_cast<uint4*>(dst + j) = lo;
              if (n + j + 8 < a.N) *reinterpret_cast<uint4*>(dst + j + 8) = hi;
            }
          }
        }
      } else {
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < 64; ++j) {
          acc[j] = silu_mul(acc[j], acc[64 + j]);  // columns beyond N are zeros
          top = max(top, __float_as_uint(fabsf(acc[j])));
        }
        // the other 64 columns of this row's block belong to the other warp of the lane quarter
        top_half[part][32 * q + lane] = top;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory");
        top = max(top, top_half[part ^ 1][32 * q + lane]);
        const float s = block_scale(__uint_as_float(top)), lift = lift_of(s);
        if (__any_sync(0xffffffffu, lift != 1.0f)) {
#pragma unroll
          for (int j = 0; j < 64; ++j) acc[j] *= lift;
        }
        const Divisor d(s * lift);
        const int n = at.n0 + 64 * part;
        if (here) {
          uint8_t* dst = a.codes + row * a.N + n;
#pragma unroll
          for (int j = 0; j < 64; j += 16) {
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float* y = acc + j + 4 * i;
              d.divide(y[0], y[1]);
              d.divide(y[2], y[3]);
              o[i] = pack4_e4m3(y[0], y[1], y[2], y[3]);
            }
            if (n + j < a.N) *reinterpret_cast<uint4*>(dst + j) = make_uint4(o[0], o[1], o[2], o[3]);
          }
          if (part == 0) a.scales[row * a.nb + at.n0 / kBlk] = s;
        }
        asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory");  // both have read before the next tile writes
      }
    }
    // rows behind the last expert's: one contiguous piece of each output
    if (a.zero_tail && a.offsets) {
      const long long from = row_start[a.E], rows = a.R - from;
      const long long me = (long long)blockIdx.x * 256 + threadIdx.x - 128, all = (long long)gridDim.x * 256;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      if constexpr (kHalves == 1) {
        uint4* dst = reinterpret_cast<uint4*>(a.c + from * a.N);
        for (long long i = me; i < rows * a.N / 8; i += all) dst[i] = zero;
      } else {
        uint4* dst = reinterpret_cast<uint4*>(a.codes + from * a.N);
        for (long long i = me; i < rows * a.N / 16; i += all) dst[i] = zero;
        for (long long i = me; i < rows * a.nb; i += all) a.scales[from * a.nb + i] = kScaleFloor;
      }
    }
  }

  // ------------------------------------------------------------ teardown (also the abort path)
  __syncwarp();
  if (*reinterpret_cast<volatile int*>(&abort_flag)) {
    const long long t0 = clock64();
    while (clock64() - t0 < 4000000LL) {
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // the pair leaves together: MMAs read both CTAs' shared memory, both share barriers
  if (warp == 2) {
    tc_fence_after_sync();
    tmem_dealloc<kCtas>(tmem, 512);
  }
}

}  // namespace fp8
}  // namespace magi
