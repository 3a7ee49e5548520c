// Rows sorted by expert, and the sums that bring them back to their tokens.
#include "ftb_lm.cuh"

#include <cooperative_groups.h>
#include <mutex>

namespace ftb {

namespace cg = cooperative_groups;

// ------------------------------------------------------------------ stable counting sort of expert ids
// One cluster does it in one launch: a CTA owns a run of rows, a warp a run of the CTA's.  Every warp counts its ids
// into a row of shared memory of its own (lanes with equal ids find each other by ballots, so nothing is added
// atomically and the result does not depend on timing), the counts are summed over warps, over the CTAs of the cluster
// (through distributed shared memory) and over the experts, and a second walk gives every row its place.  Bytes: ids
// twice (the second time from L2), order once, slots three times; bound by latency up to some ten thousand rows (device time,
// in a graph: 64 rows of 64 experts 2.6 us, 4000 of 16 3.4, 16384 of 32 5.7, 32768 of 256 10.2), then by the scattered
// stores of eight SMs (262144 rows of 256: 49 us, beside products of milliseconds).
constexpr int kPlanCtas = 8;

// Lanes with the same key (`bits` of it): one ballot per bit.
__device__ __forceinline__ unsigned same_key(int key, int bits) {
  unsigned same = 0xffffffffu;
  for (int b = 0; b < bits; ++b) {
    const bool one = (key >> b) & 1;
    const unsigned ones = __ballot_sync(0xffffffffu, one);
    same &= one ? ones : ~ones;
  }
  return same;
}

__global__ void __launch_bounds__(1024) expert_plan_kernel(const int* __restrict__ ids, int* __restrict__ offsets,
                                                           int* __restrict__ order, int* slots, int rows,
                                                           int experts) {
  extern __shared__ int smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* hist = smem;                      // [warps][experts]
  int* total = hist + warps * experts;   // [experts] this CTA's count
  int* start = total + experts;          // [experts] place of this CTA's first row of an expert
  __shared__ int placed;                 // rows of all experts
  const long long per_warp = ((static_cast<long long>(rows) + ctas * warps - 1) / (ctas * warps) + 31) / 32 * 32;
  const long long r0 = (static_cast<long long>(rank) * warps + warp) * per_warp;
  const long long r1 = min(r0 + per_warp, static_cast<long long>(rows));
  const int bits = 32 - __clz(experts);  // of keys 0..experts, the last standing for dropped rows
  int* mine = hist + warp * experts;
  for (int e = lane; e < experts; e += 32) mine[e] = 0;
  __syncwarp();
  grid_dependency_wait();
  grid_launch_dependents();
  auto id_of = [&](long long row) {
    const int key = row < r1 ? ids[row] : experts;
    return key < 0 || key > experts ? experts : key;
  };
  // A row's number among its warp's rows of the same expert waits in `slots` for the second walk, which then has no
  // order to keep; the next ids are on their way meanwhile.
  int next = id_of(r0 + lane);
  for (long long r = r0; r < r1; r += 32) {
    const int key = next;
    next = id_of(r + 32 + lane);
    const unsigned same = same_key(key, bits);
    const int before = key < experts ? mine[key] : 0;
    if (r + lane < r1) slots[r + lane] = before + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (key < experts && lane == __ffs(same) - 1) mine[key] = before + __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += blockDim.x) {
    int run = 0;
    for (int w = 0; w < warps; ++w) {
      const int c = hist[w * experts + e];
      hist[w * experts + e] = run;
      run += c;
    }
    total[e] = run;
  }
  cluster.sync();
  // counts of all CTAs, and of those before this one
  for (int e = threadIdx.x; e < experts; e += blockDim.x) {
    int before = 0, all = 0, v[kPlanCtas];
#pragma unroll
    for (int c = 0; c < kPlanCtas; ++c) v[c] = c < ctas ? cluster.map_shared_rank(total, c)[e] : 0;
#pragma unroll
    for (int c = 0; c < kPlanCtas; ++c) {
      if (c < rank) before += v[c];
      all += v[c];
    }
    start[e] = before;
    // the total over CTAs goes where the warps' scan below finds it; own total is not needed any more once every CTA
    // has read it, which the next cluster barrier says
    hist[warps * experts + 2 * experts + e] = all;
  }
  cluster.sync();
  if (warp == 0) {
    const int* all = hist + warps * experts + 2 * experts;
    int base = 0;
    for (int e0 = 0; e0 < experts; e0 += 32) {
      const int v = e0 + lane < experts ? all[e0 + lane] : 0;
      int x = v;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      if (e0 + lane < experts) {
        start[e0 + lane] += base + x - v;
        if (rank == 0) offsets[e0 + lane] = base + x - v;
      }
      base += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) {
      placed = base;
      if (rank == 0) offsets[experts] = base;
    }
  }
  __syncthreads();
#pragma unroll 4
  for (long long row = r0 + lane; row < r1; row += 32) {
    const int key = id_of(row);
    const int place = key < experts ? start[key] + mine[key] + slots[row] : -1;
    slots[row] = place;
    if (place >= 0) order[place] = static_cast<int>(row);
  }
  for (long long q = placed + static_cast<long long>(rank) * blockDim.x + threadIdx.x; q < rows;
       q += static_cast<long long>(ctas) * blockDim.x)
    order[q] = -1;
}

static int launch_plan(const int* ids, int* offsets, int* order, int* slots, int64_t rows, int64_t experts,
                       cudaStream_t stream) {
  // one CTA up to 1024 rows (32 rows a warp); above that eight share them (4000 rows: 3.4 us, in one 10.3)
  const int ctas = rows > 1024 ? kPlanCtas : 1;
  int64_t warps = ceil_div64(rows, static_cast<int64_t>(ctas) * 32);
  if (warps < 4) warps = 4;
  if (warps > 32) warps = 32;
  const size_t smem = static_cast<size_t>(warps + 3) * experts * sizeof(int);
  static std::mutex mu;
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 0 && dev < 64 && !done[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(expert_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 35 * FTB_MAX_EXPERTS * static_cast<int>(sizeof(int)));
      if (e != cudaSuccess) return launch_status(e);
      done[dev] = true;
    }
  }
  return launch_overlapped(expert_plan_kernel, dim3(static_cast<unsigned>(ctas)), dim3(static_cast<unsigned>(warps * 32)), smem,
                           ctas, stream, ids, offsets, order, slots, static_cast<int>(rows), static_cast<int>(experts));
}

// ------------------------------------------------------------------ weighted sum of a token's rows
// Bound by reading y once; a thread owns VEC neighbouring columns of one token and adds its rows in slot order in fp32.
// (The rows themselves are 16-bit tensors of the caller, rounded once when expert_linear stored them: half the bytes of both
// kernels, for a second rounding in the result, 2.0e-3 against 64 bits instead of 1.6e-3 over both.)
// 4096 tokens x 4 rows x 2048 with residual: 16.8 us, 5.7 TB/s, 0.87 of the measured copy rate.
template <int VEC>
__global__ void __launch_bounds__(128)
expert_combine_kernel(const uint16_t* __restrict__ y, const int* __restrict__ slots, const float* __restrict__ weights,
                      const uint16_t* residual, uint16_t* out, int top_k, long long n, long long rows, int blocks_n,
                      int f16_i) {
  grid_dependency_wait();
  grid_launch_dependents();
  const bool f16 = f16_i != 0;
  const long long t = blockIdx.x / blocks_n;
  const long long c = (static_cast<long long>(blockIdx.x % blocks_n) * 128 + threadIdx.x) * VEC;
  if (c >= n) return;
  float acc[VEC] = {};
  if (residual) {
    if constexpr (VEC == 8) {
      const uint4 q = *reinterpret_cast<const uint4*>(residual + t * n + c);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack16(w[i], f16);
        acc[2 * i] = f.x;
        acc[2 * i + 1] = f.y;
      }
    } else {
      acc[0] = from16(residual[t * n + c], f16);
    }
  }
  // four rows on their way at a time, added in slot order
  const int* slot = slots + t * top_k;
  for (int j0 = 0; j0 < top_k; j0 += 4) {
    float w[4];
    uint4 q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int place = j0 + e < top_k ? slot[j0 + e] : -1;
      const bool there = place >= 0 && place < rows;
      w[e] = !there ? 0.0f : weights ? weights[t * top_k + j0 + e] : 1.0f;
      q[e] = make_uint4(0, 0, 0, 0);
      if constexpr (VEC == 8) {
        if (there) q[e] = *reinterpret_cast<const uint4*>(y + place * n + c);
      } else {
        if (there) q[e].x = y[place * n + c];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (VEC == 8) {
        const uint32_t v[4] = {q[e].x, q[e].y, q[e].z, q[e].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack16(v[i], f16);
          acc[2 * i] = fmaf(w[e], f.x, acc[2 * i]);
          acc[2 * i + 1] = fmaf(w[e], f.y, acc[2 * i + 1]);
        }
      } else {
        acc[0] = fmaf(w[e], from16(static_cast<uint16_t>(q[e].x), f16), acc[0]);
      }
    }
  }
  if constexpr (VEC == 8) {
    *reinterpret_cast<uint4*>(out + t * n + c) =
        make_uint4(pack16(acc[0], acc[1], f16), pack16(acc[2], acc[3], f16), pack16(acc[4], acc[5], f16), pack16(acc[6], acc[7], f16));
  } else {
    out[t * n + c] = to16(acc[0], f16);
  }
}

// One warp per row: dy of its place and the row's dot product, whose lane sums meet in a fixed tree.  Bound by y and dy; the
// token's dout comes from L2 after its first row.  4096 tokens x 4 rows x 2048, a sixteenth of them dropped: both results
// 29.1 us, 4.9 TB/s, 0.75 of the copy rate; dy alone 23.4, dweights alone 15.9.
template <int VEC>
__global__ void __launch_bounds__(256)
expert_combine_backward_kernel(const uint16_t* __restrict__ dout, const uint16_t* __restrict__ y,
                               const int* __restrict__ slots, const float* __restrict__ weights, uint16_t* __restrict__ dy,
                               float* __restrict__ dweights, long long rows, int top_k, long long n, int f16_i) {
  grid_dependency_wait();
  grid_launch_dependents();
  const bool f16 = f16_i != 0;
  const long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const int place = slots[row];
  const bool live = place >= 0 && place < rows;
  float dot = 0.0f;
  if (live) {
    const float w = weights ? weights[row] : 1.0f;
    const uint16_t* g = dout + row / top_k * n;
    for (long long c = static_cast<long long>(lane) * VEC; c < n; c += 32 * VEC) {
      if constexpr (VEC == 8) {
        const uint4 q = *reinterpret_cast<const uint4*>(g + c);
        const uint32_t gv[4] = {q.x, q.y, q.z, q.w};
        uint32_t o[4];
        uint4 qy = make_uint4(0, 0, 0, 0);
        if (dweights) qy = *reinterpret_cast<const uint4*>(y + place * n + c);
        const uint32_t yv[4] = {qy.x, qy.y, qy.z, qy.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 a = unpack16(gv[i], f16), b = unpack16(yv[i], f16);
          o[i] = pack16(w * a.x, w * a.y, f16);
          dot = fmaf(a.x, b.x, dot);
          dot = fmaf(a.y, b.y, dot);
        }
        if (dy) *reinterpret_cast<uint4*>(dy + place * n + c) = make_uint4(o[0], o[1], o[2], o[3]);
      } else {
        const float a = from16(g[c], f16);
        if (dweights) dot = fmaf(a, from16(y[place * n + c], f16), dot);
        if (dy) dy[place * n + c] = to16(w * a, f16);
      }
    }
  }
  if (!dweights) return;
#pragma unroll
  for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
  if (lane == 0) dweights[row] = dot;
}

static bool vec_ok(int64_t n, const void* a, const void* b, const void* c) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c);
  return n % 8 == 0 && (all & 15) == 0;
}

static int combine_checks(int dtype, int64_t tokens, int64_t top_k, int64_t n) {
  if (dtype != FTB_BF16 && dtype != FTB_F16) return FTB_E_BAD_ARG;
  if (tokens < 0 || top_k <= 0 || n <= 0) return FTB_E_BAD_ARG;
  if (top_k > FTB_MAX_TOP_K || tokens > (1ll << 30) / top_k || n > (1ll << 30)) return FTB_E_TOO_LARGE;
  return FTB_OK;
}

}  // namespace ftb

extern "C" {

int ftb_expert_plan(const int32_t* ids, int32_t* offsets, int32_t* order, int32_t* slots, int64_t rows, int64_t experts,
                    void* stream) {
  using namespace ftb;
  if (rows < 0 || experts <= 0 || !offsets) return FTB_E_BAD_ARG;
  if (rows > 0 && (!ids || !order || !slots)) return FTB_E_BAD_ARG;
  if (experts > FTB_MAX_EXPERTS || rows > (1ll << 30)) return FTB_E_TOO_LARGE;
  const int rc = device_ok();
  if (rc) return rc;
  return launch_plan(ids, offsets, order, slots, rows, experts, static_cast<cudaStream_t>(stream));
}

int ftb_expert_combine(int dtype, const void* y, const int32_t* slots, const float* weights, const void* residual,
                       void* out, int64_t tokens, int64_t top_k, int64_t n, void* stream) {
  using namespace ftb;
  int rc = combine_checks(dtype, tokens, top_k, n);
  if (rc) return rc;
  if (tokens == 0) return FTB_OK;
  if (!y || !slots || !out) return FTB_E_BAD_ARG;
  rc = device_ok();
  if (rc) return rc;
  const bool vec = vec_ok(n, y, residual, out);
  const int64_t blocks_n = ceil_div64(n, vec ? 1024 : 128);
  if (blocks_n * tokens > 0x7fffffff) return FTB_E_TOO_LARGE;
  const unsigned grid = static_cast<unsigned>(blocks_n * tokens);
  const uint16_t* yv = static_cast<const uint16_t*>(y);
  const uint16_t* rv = static_cast<const uint16_t*>(residual);
  uint16_t* ov = static_cast<uint16_t*>(out);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int k = static_cast<int>(top_k), f16 = dtype == FTB_F16;
  return launch_overlapped(vec ? expert_combine_kernel<8> : expert_combine_kernel<1>, dim3(grid), dim3(128), 0, 1, s, yv, slots,
                           weights, rv, ov, k, n, tokens * top_k, static_cast<int>(blocks_n), f16);
}

int ftb_expert_combine_backward(int dtype, const void* dout, const void* y, const int32_t* slots, const float* weights,
                                void* dy, float* dweights, int64_t tokens, int64_t top_k, int64_t n, void* stream) {
  using namespace ftb;
  int rc = combine_checks(dtype, tokens, top_k, n);
  if (rc) return rc;
  if (tokens == 0) return FTB_OK;
  if (!dy && !dweights) return FTB_E_BAD_ARG;
  if (!dout || !slots || (dweights && !y)) return FTB_E_BAD_ARG;
  rc = device_ok();
  if (rc) return rc;
  const int64_t rows = tokens * top_k;
  const unsigned grid = static_cast<unsigned>(ceil_div64(rows, 8));
  const uint16_t* g = static_cast<const uint16_t*>(dout);
  const uint16_t* yv = static_cast<const uint16_t*>(y);
  uint16_t* d = static_cast<uint16_t*>(dy);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int k = static_cast<int>(top_k), f16 = dtype == FTB_F16;
  const bool vec = vec_ok(n, dout, dweights ? y : nullptr, dy);
  return launch_overlapped(vec ? expert_combine_backward_kernel<8> : expert_combine_backward_kernel<1>, dim3(grid), dim3(256), 0, 1,
                           s, g, yv, slots, weights, d, dweights, rows, k, n, f16);
}

}  // extern "C"
