// Device code of the routed (mixture-of-experts) row movements: tokens sorted by expert, gathered into expert order (bf16,
// or quantised to block-scaled fp8 on the way), added up again with the router's weights, and the gradients of both.
//
//   slot s = t * k + j        the j-th expert choice of token t
//   row_slot[r] = s           which slot sorted row r holds (-1: none, a row behind the last expert's)
//   slot_row[s] = r           where slot s went (-1: the slot has no expert)
//
// All of them are bound by HBM: the arithmetic is a few operations per byte.  What counts is that every token row is
// read ONCE however many experts it goes to (the kernels walk tokens, not sorted rows), that accesses are 16 bytes wide
// and contiguous per row, and that a call is one launch.  Indices read from memory are bounds-checked: one that is out of
// range counts as "no expert", so a bad index array gives wrong rows but no access outside the operands.
// Every kernel may be scheduled while the previous one drains and waits for it before its first access to global memory
// (gather of 8192 rows of 4096 for two experts each 35.5 to 34.4 us back to back, quantiser of 8192 x 4096 17.7 to 17.4,
// of 2005 x 2064 for eight experts 9.05 to 8.55).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "fp8_format.cuh"
#include "ptx_sm100.cuh"

namespace magi {

constexpr int kMaxExperts = 1024;   // one 32-warp histogram of 1025 counters is 131 KB of shared memory
constexpr int kSlotBatch = 4;       // expert rows of one token in flight per thread of the combine's backward

// ---------------------------------------------------------------- sort
// Stable counting sort of the slots by expert, slots without an expert last.  One thread-block cluster does it in one
// launch: each warp owns a contiguous range of slots and a histogram row; equal keys inside a warp step are ranked by lane,
// so ties keep slot order and no atomic decides anything.  The CTAs of the cluster read each other's totals
// through distributed shared memory.  hist: [warps][E + 1], total: [E + 1], start: [E + 1].
constexpr int kSortCtas = 16;  // more than the 8 every GPU has to offer: asked for, with 8 to fall back on
constexpr int kSortKeep = 4;  // steps of 32 slots whose keys and matches a warp keeps between its two passes

__device__ __forceinline__ int ld_cluster_s32(uint32_t cluster_addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(cluster_addr));
  return v;
}

__device__ __forceinline__ int slot_key(const void* ids, int wide, int s, int end, int E) {
  if (s >= end) return E + 1;  // no slot: equal to other absent lanes only
  const long long v = wide ? static_cast<const long long*>(ids)[s] : (long long)static_cast<const int*>(ids)[s];
  return (v >= 0 && v < E) ? (int)v : E;
}

// Lanes whose key (below 2^bits) equals mine: one vote per bit of the key.  (__match_any_sync walks the distinct keys one
// by one: with 128 experts a step took about 500 cycles.)
__device__ __forceinline__ unsigned equal_lanes(int key, int bits) {
  unsigned m = 0xffffffffu;
#pragma unroll
  for (int b = 0; b < 11; ++b) {  // kMaxExperts + 1 has 11 bits
    if (b >= bits) break;
    const bool one = (key >> b) & 1;
    const unsigned votes = __ballot_sync(0xffffffffu, one);
    m &= one ? votes : ~votes;
  }
  return m;
}

__global__ void __launch_bounds__(1024, 1)
expert_sort_kernel(const void* ids, int wide, int R, int E, int* row_slot, int* slot_row, int* offsets, int ctas) {
  extern __shared__ int sort_smem[];
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned lower = (1u << lane) - 1u;
  const int bits = 32 - __clz(E + 1);
  const int buckets = E + 1;
  int* hist = sort_smem + warp * buckets;
  int* total = sort_smem + warps * buckets;
  int* all = total + buckets;
  int* before = all + buckets;
  const int rank = ctas > 1 ? (int)cluster_ctarank() : 0;

  // a warp's share, a multiple of 32 slots
  const int units = ctas * warps;
  const long long share = (((long long)R + units - 1) / units + 31) / 32 * 32;
  const long long first = share * (rank * warps + warp);
  const int lo = (int)(first < R ? first : R), hi = (int)(first + share < R ? first + share : R);

  for (int i = threadIdx.x; i < warps * buckets; i += blockDim.x) sort_smem[i] = 0;
  grid_launch_dependents();
  grid_dependency_wait();
  // the first steps' keys and matches stay in registers for the second pass
  int key[kSortKeep];
  unsigned same[kSortKeep];
#pragma unroll
  for (int i = 0; i < kSortKeep; ++i) key[i] = slot_key(ids, wide, lo + 32 * i + lane, hi, E);
  __syncthreads();
  auto count = [&](int k, unsigned m) {  // the lowest lane of each group of equal keys
    if (k <= E && (m & lower) == 0) hist[k] += __popc(m);
    __syncwarp();
  };
#pragma unroll
  for (int i = 0; i < kSortKeep; ++i) {
    same[i] = 0;
    if (lo + 32 * i < hi) {
      same[i] = equal_lanes(key[i], bits);
      count(key[i], same[i]);
    }
  }
  for (int s = lo + 32 * kSortKeep; s < hi; s += 32) {
    const int k = slot_key(ids, wide, s + lane, hi, E);
    count(k, equal_lanes(k, bits));
  }
  __syncthreads();
  // histogram column e -> exclusive prefix over this CTA's warps, and the CTA's total
  for (int e = threadIdx.x; e < buckets; e += blockDim.x) {
    int sum = 0;
    for (int w = 0; w < warps; ++w) {
      const int n = sort_smem[w * buckets + e];
      sort_smem[w * buckets + e] = sum;
      sum += n;
    }
    total[e] = sum;
  }
  __syncthreads();
  if (ctas > 1) cluster_sync_all();
  for (int e = threadIdx.x; e < buckets; e += blockDim.x) {
    int sum = 0, low = 0;
    if (ctas == 1) {
      sum = total[e];
    } else {
      const uint32_t at = smem_u32(total + e);
#pragma unroll
      for (int c = 0; c < kSortCtas; ++c)
        if (c < ctas) {
          const int n = ld_cluster_s32(map_to_cta(at, c));
          low += c < rank ? n : 0;
          sum += n;
        }
    }
    all[e] = sum;
    before[e] = low;
  }
  __syncthreads();
  if (warp == 0) {  // first row of each bucket
    int carry = 0;
    for (int b = 0; b < buckets; b += 32) {
      const int e = b + lane;
      const int n = e < buckets ? all[e] : 0;
      int scan = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d) scan += up;
      }
      if (e < buckets) {
        const int first = carry + scan - n;
        all[e] = first + before[e];
        if (rank == 0) offsets[e] = first;  // offsets[E] = first row without an expert
      }
      carry += __shfl_sync(0xffffffffu, scan, 31);
    }
  }
  __syncthreads();
  auto place = [&](int s, int k, unsigned m) {
    const int base = k <= E ? hist[k] : 0;
    __syncwarp();
    if (k <= E) {
      if ((m & lower) == 0) hist[k] = base + __popc(m);
      const int r = all[k] + base + __popc(m & lower);
      row_slot[r] = k < E ? s : -1;
      slot_row[s] = k < E ? r : -1;
    }
    __syncwarp();
  };
#pragma unroll
  for (int i = 0; i < kSortKeep; ++i)
    if (lo + 32 * i < hi) place(lo + 32 * i + lane, key[i], same[i]);
  for (int s = lo + 32 * kSortKeep; s < hi; s += 32) {
    const int k = slot_key(ids, wide, s + lane, hi, E);
    place(s + lane, k, equal_lanes(k, bits));
  }
  if (ctas > 1) cluster_sync_all();  // nobody leaves while its totals may still be read
}

// ---------------------------------------------------------------- row movement
// Thread (x, y) of block b: token (b / col_chunks) * blockDim.y + y, 16-byte column piece (b % col_chunks) * blockDim.x + x.
struct RowPiece {
  long long t;
  int c;
};
__device__ __forceinline__ RowPiece row_piece(int col_chunks) {
  RowPiece p;
  p.t = (long long)(blockIdx.x / col_chunks) * blockDim.y + threadIdx.y;
  p.c = (blockIdx.x % col_chunks) * blockDim.x + threadIdx.x;
  return p;
}
// Whether row s holds no slot.
__device__ __forceinline__ bool empty_row(const int* row_slot, long long s, long long R) {
  const int slot = row_slot[s];
  return slot < 0 || slot >= R;
}
// A load of data that is used once.  Volatile, so that it stays behind grid_dependency_wait (the compiler may move a
// read-only load or the intrinsic in front of it).
__device__ __forceinline__ uint4 ld_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// xs[slot_row[t, j]] = x[t]; row t * k + j is zeroed when it holds no slot.
__global__ void __launch_bounds__(256)
expert_gather_kernel(const uint4* x, long long ldx, const int* row_slot, const int* slot_row, uint4* xs, long long T, int k,
                     int vecs, int col_chunks) {
  grid_launch_dependents();
  grid_dependency_wait();
  const RowPiece p = row_piece(col_chunks);
  if (p.t >= T || p.c >= vecs) return;
  const long long R = T * k;
  const uint4 v = ld_stream(x + p.t * ldx + p.c);
  for (int j = 0; j < k; ++j) {
    const long long s = p.t * k + j;
    const int r = slot_row[s];
    if (r >= 0 && r < R) xs[(long long)r * vecs + p.c] = v;
    if (empty_row(row_slot, s, R)) xs[s * vecs + p.c] = make_uint4(0, 0, 0, 0);
  }
}

__device__ __forceinline__ void bf16x8_to_f32(uint4 v, float (&f)[8]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(u[i] << 16);
    f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 f32_to_bf16x8(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

// out[t] = sum over j of w[t, j] * y[slot_row[t, j]] in fp32, j ascending, one rounding; w null: all ones (the gradient of
// the gather).  Slots without an expert add nothing, whatever their weight.  A thread keeps kSlots * kPieces loads of 16
// bytes in flight: kSlots rows of its token, kPieces column pieces a block's width apart (8192 tokens of k = 2, H = 4096: two
// loads 67 us, eight 40 us, eight with three blocks an SM 36 us).
template <int kSlots, int kPieces>
__global__ void __launch_bounds__(256, 3)
expert_combine_kernel(const uint4* y, long long ldy, const float* w, const int* slot_row, uint4* out, long long T, int k,
                      int vecs, int col_chunks) {
  grid_launch_dependents();
  grid_dependency_wait();
  const long long t = (long long)(blockIdx.x / col_chunks) * blockDim.y + threadIdx.y;
  const int c0 = (blockIdx.x % col_chunks) * blockDim.x * kPieces + threadIdx.x;
  if (t >= T) return;
  const long long R = T * k;
  float acc[kPieces][8];
#pragma unroll
  for (int p = 0; p < kPieces; ++p)
#pragma unroll
    for (int q = 0; q < 8; ++q) acc[p][q] = 0.0f;
  for (int j0 = 0; j0 < k; j0 += kSlots) {
    uint4 v[kSlots][kPieces];
    float wj[kSlots];
    int r[kSlots];
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const long long s = t * k + j0 + i;
      r[i] = j0 + i < k ? slot_row[s] : -1;
      if (r[i] >= R) r[i] = -1;
      wj[i] = (r[i] >= 0 && w) ? w[s] : 1.0f;
    }
#pragma unroll
    for (int i = 0; i < kSlots; ++i)
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        const int c = c0 + p * blockDim.x;
        if (r[i] >= 0 && c < vecs) v[i][p] = ld_stream(y + (long long)r[i] * ldy + c);
      }
#pragma unroll
    for (int i = 0; i < kSlots; ++i)
#pragma unroll
      for (int p = 0; p < kPieces; ++p)
        if (r[i] >= 0 && c0 + p * (int)blockDim.x < vecs) {
          float f[8];
          bf16x8_to_f32(v[i][p], f);
#pragma unroll
          for (int q = 0; q < 8; ++q) acc[p][q] = fmaf(wj[i], f[q], acc[p][q]);
        }
  }
#pragma unroll
  for (int p = 0; p < kPieces; ++p) {
    const int c = c0 + p * blockDim.x;
    if (c < vecs) out[t * vecs + c] = f32_to_bf16x8(acc[p]);
  }
}

// The combine's gradients in one pass: dy[slot_row[t, j]] = w[t, j] * dout[t] (rows without a slot are zeroed) and
// dw[t, j] = <dout[t], y[slot_row[t, j]]> (0 for a slot without an expert), sums in fp32 in a fixed order.
// token_warps warps (1, 2, 4 or 8) share a token.  dy or dw may be null (y is not read without dw).  Batches of four rows
// and four blocks an SM: 8192 tokens x 8 rows of 2048, back to back, 100 us; of eight rows and two blocks 136 us.
__global__ void __launch_bounds__(256, 4)
expert_combine_backward_kernel(const uint4* dout, long long lddout, const uint4* y, long long ldy, const float* w,
                               const int* row_slot, const int* slot_row, uint4* dy, float* dw, long long T, int k, int vecs,
                               int token_warps) {
  __shared__ float red[8][kSlotBatch];
  grid_launch_dependents();
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp % token_warps;
  const long long t = (long long)blockIdx.x * (8 / token_warps) + warp / token_warps;
  const bool here = t < T;
  const long long R = T * k;
  const int step = token_warps * 32;
  for (int j0 = 0; j0 < k; j0 += kSlotBatch) {
    float dot[kSlotBatch], wj[kSlotBatch];
    int r[kSlotBatch];
    unsigned empty = 0;  // bit i: row t * k + j0 + i holds no slot
#pragma unroll
    for (int i = 0; i < kSlotBatch; ++i) {
      const long long s = t * k + j0 + i;
      const bool on = here && j0 + i < k;
      dot[i] = 0.0f;
      r[i] = on ? slot_row[s] : -1;
      if (r[i] >= R) r[i] = -1;
      wj[i] = (r[i] >= 0 && dy) ? w[s] : 0.0f;
      if (on && dy && empty_row(row_slot, s, R)) empty |= 1u << i;
    }
    if (here)
      for (int c = part * 32 + lane; c < vecs; c += step) {
        float d[8];
        uint4 v[kSlotBatch];
        const uint4 dv = dout[t * lddout + c];
        if (dw) {
#pragma unroll
          for (int i = 0; i < kSlotBatch; ++i)
            if (r[i] >= 0) v[i] = ld_stream(y + (long long)r[i] * ldy + c);
        }
        bf16x8_to_f32(dv, d);
#pragma unroll
        for (int i = 0; i < kSlotBatch; ++i) {
          if (dw && r[i] >= 0) {
            float f[8];
            bf16x8_to_f32(v[i], f);
#pragma unroll
            for (int q = 0; q < 8; ++q) dot[i] = fmaf(d[q], f[q], dot[i]);
          }
          if (dy && r[i] >= 0) {
            float f[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) f[q] = wj[i] * d[q];
            dy[(long long)r[i] * vecs + c] = f32_to_bf16x8(f);
          }
          if (empty >> i & 1u) dy[(t * k + j0 + i) * vecs + c] = make_uint4(0, 0, 0, 0);
        }
      }
    if (dw) {
#pragma unroll
      for (int i = 0; i < kSlotBatch; ++i)
#pragma unroll
        for (int o = 16; o; o >>= 1) dot[i] += __shfl_xor_sync(0xffffffffu, dot[i], o);
      if (lane == 0)
#pragma unroll
        for (int i = 0; i < kSlotBatch; ++i) red[warp][i] = dot[i];
      __syncthreads();
      if (here && part == 0 && lane < kSlotBatch && j0 + lane < k) {
        float sum = 0.0f;
        for (int q = 0; q < token_warps; ++q) sum += red[warp + q][lane];
        dw[t * k + j0 + lane] = sum;
      }
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------- block quantiser
// Per row and 128 columns: s = max(max|x| / 448, 2^-126), q = e4m3(x / s).  Eight lanes hold a block (16 columns each).
// The maximum is taken on the bf16 bit patterns without their sign, which order like the values and put infinities and
// NaN on top: a block with an infinity gets s = inf (its finite elements become 0, the infinity NaN), one with a NaN is
// all NaN.  Codes and scales equal the formula evaluated in fp32 with IEEE divisions bit for bit (the tests compare them for
// every pair of bf16 mantissas of x and of the block's maximum): the quotient is a corrected product (fp8_format.cuh), and
// blocks with an extreme or non-finite scale, where the correction is not exact, divide.  8192 x 4096:
// the bytes take 15.5 us; with sixteen divisions a thread 26.6 us, with the correction 18.9 us, with two values an
// instruction 17.7 us.
// slot_row null: codes[t], scales[t] from x[t].  Else the quantised gather: token t goes to rows slot_row[t, j] and row
// t * k + j gets zero codes and the floor scale when it holds no slot.
__global__ void __launch_bounds__(256)
quantize_fp8_block_kernel(const uint4* x, long long ldx, const int* row_slot, const int* slot_row, uint4* codes,
                          float* scales, long long T, int k, int pieces, int col_chunks, int kb) {
  grid_launch_dependents();
  grid_dependency_wait();
  const RowPiece p = row_piece(col_chunks);
  const bool on = p.t < T && p.c < pieces;
  uint4 a = make_uint4(0, 0, 0, 0), b = a;
  if (on) {
    a = ld_stream(x + p.t * ldx + 2 * p.c);
    b = ld_stream(x + p.t * ldx + 2 * p.c + 1);
  }
  const uint32_t m = 0x7fff7fffu;
  uint32_t top = __vmaxu2(__vmaxu2(__vmaxu2(a.x & m, a.y & m), __vmaxu2(a.z & m, a.w & m)),
                          __vmaxu2(__vmaxu2(b.x & m, b.y & m), __vmaxu2(b.z & m, b.w & m)));
  top = max(top & 0xffffu, top >> 16);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float s = block_scale(__uint_as_float(top << 16));
  if (!on) return;
  float f[8], g[8];
  bf16x8_to_f32(a, f);
  bf16x8_to_f32(b, g);
  if (s > kScaleSmall && s < kScaleLarge) {
    const Divisor d(s);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      d.divide(f[i], f[i + 1]);
      d.divide(g[i], g[i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[i] = __fdiv_rn(f[i], s);
      g[i] = __fdiv_rn(g[i], s);
    }
  }
  const uint4 q = make_uint4(pack4_e4m3(f[0], f[1], f[2], f[3]), pack4_e4m3(f[4], f[5], f[6], f[7]),
                             pack4_e4m3(g[0], g[1], g[2], g[3]), pack4_e4m3(g[4], g[5], g[6], g[7]));
  const bool writes_scale = (p.c & 7) == 0;
  if (!slot_row) {
    codes[p.t * pieces + p.c] = q;
    if (writes_scale) scales[p.t * kb + (p.c >> 3)] = s;
    return;
  }
  const long long R = T * k;
  for (int j = 0; j < k; ++j) {
    const long long sl = p.t * k + j;
    const int r = slot_row[sl];
    if (r >= 0 && r < R) {
      codes[(long long)r * pieces + p.c] = q;
      if (writes_scale) scales[(long long)r * kb + (p.c >> 3)] = s;
    }
    if (empty_row(row_slot, sl, R)) {
      codes[sl * pieces + p.c] = make_uint4(0, 0, 0, 0);
      if (writes_scale) scales[sl * kb + (p.c >> 3)] = kScaleFloor;
    }
  }
}

}  // namespace magi
