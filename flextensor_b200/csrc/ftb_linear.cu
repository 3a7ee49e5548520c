// Host side of the products with an epilogue (ftb_linear, ftb_expert_linear and their gradients) and the elementwise
// kernels of the backward pass.
#include "ftb_linear.h"

namespace ftb {

// ------------------------------------------------------------------ dz = dy * act'(z), and the sums for db
// One pass over dy and z, bound by those bytes: a thread owns VEC neighbouring columns (16-byte accesses for VEC = 8)
// and walks the rows of its chunk; the eight rows of a block are added through shared memory and every chunk leaves
// one row of fp32 partial sums, which bias_sum_kernel adds in chunk order, so db does not depend on timing.
// db alone (no dz): 4096 x 4096 with tanh GELU 24.1 us, with erf GELU 27.1, without activation 14.3; 4000 x (2 x 1400) gated
// SiLU 17.1; with dz in front of dx instead: 22 and 26 us at 4096 x 4096, 4.2 TB/s.
// dz is rounded once to the element type, because the products that read it take 16-bit operands: two halves of it (high
// and low) would double their MMAs and bytes.  It costs their results a second rounding of the operands' own size (error
// against 64 bits 2.3e-3 instead of 1.7e-3 in bf16, 2.9e-4 instead of 2.1e-4 in fp16); db is summed before it.
constexpr int kDzRows = 8;

template <int VEC>
struct DzIn {
  uint32_t d[(VEC + 1) / 2], a[(VEC + 1) / 2], u[(VEC + 1) / 2];
};

template <int VEC>
__device__ __forceinline__ void dz_read(uint32_t (&w)[(VEC + 1) / 2], const uint16_t* p) {
  if constexpr (VEC == 8) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    w[0] = q.x;
    w[1] = q.y;
    w[2] = q.z;
    w[3] = q.w;
  } else {
    w[0] = *p;
  }
}
template <int VEC>
__device__ __forceinline__ void dz_unpack(float (&f)[VEC], const uint32_t (&w)[(VEC + 1) / 2], bool f16) {
  if constexpr (VEC == 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = unpack16(w[i], f16);
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  } else {
    f[0] = from16(static_cast<uint16_t>(w[0]), f16);
  }
}
template <int VEC>
__device__ __forceinline__ void dz_write(uint16_t* p, const float (&f)[VEC], bool f16) {
  if constexpr (VEC == 8)
    *reinterpret_cast<uint4*>(p) = make_uint4(pack16(f[0], f[1], f16), pack16(f[2], f[3], f16), pack16(f[4], f[5], f16), pack16(f[6], f[7], f16));
  else
    *p = to16(f[0], f16);
}

template <int VEC, bool GATED>
__global__ void __launch_bounds__(256)
linear_dz_kernel(const uint16_t* __restrict__ dy, const uint16_t* __restrict__ z, uint16_t* __restrict__ dz,
                 long long ldz, float* __restrict__ partial, const int* __restrict__ offsets, long long rows, long long n,
                 int act, int f16_i, int chunks) {
  const bool f16 = f16_i != 0;
  __shared__ float sums[kDzRows][32 * VEC + 1];
  grid_dependency_wait();
  grid_launch_dependents();
  const int g = blockIdx.z;
  int lo = 0, hi = static_cast<int>(rows);
  if (offsets) group_range(offsets, g, rows, &lo, &hi);
  const int per = (hi - lo + chunks - 1) / chunks;
  const long long r0 = lo + static_cast<long long>(blockIdx.y) * per;
  const long long r1 = min(r0 + per, static_cast<long long>(hi));
  const long long c0 = (static_cast<long long>(blockIdx.x) * 32 + threadIdx.x) * VEC;
  const long long wide = GATED ? 2 * n : n;
  float s0[VEC] = {}, s1[VEC] = {};
  if (c0 < n) {
    // the next row is on its way while this one is worked on
    DzIn<VEC> next;
    auto fetch = [&](long long r) {
      dz_read<VEC>(next.d, dy + r * n + c0);
      if (z) {
        dz_read<VEC>(next.a, z + r * wide + c0);
        if (GATED) dz_read<VEC>(next.u, z + r * wide + n + c0);
      }
    };
    long long r = r0 + threadIdx.y;
    if (r < r1) fetch(r);
    for (; r < r1; r += kDzRows) {
      const DzIn<VEC> in = next;
      if (r + kDzRows < r1) fetch(r + kDzRows);
      float d[VEC], g0[VEC];
      dz_unpack<VEC>(d, in.d, f16);
      if (z) {
        float a[VEC], value[VEC], slope[VEC];
        dz_unpack<VEC>(a, in.a, f16);
        act_both<VEC>(a, value, slope, act);
        if constexpr (GATED) {
          float u[VEC];
          dz_unpack<VEC>(u, in.u, f16);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            g0[i] = d[i] * u[i] * slope[i];
            value[i] *= d[i];
            s1[i] += value[i];
          }
          if (dz) dz_write<VEC>(dz + r * ldz + n + c0, value, f16);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) g0[i] = d[i] * slope[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) g0[i] = d[i];
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) s0[i] += g0[i];
      if (dz) dz_write<VEC>(dz + r * ldz + c0, g0, f16);  // one rounding to the element type: what the products read
    }
  }
  if (!partial) return;
  float* row = partial + (static_cast<long long>(g) * chunks + blockIdx.y) * wide;
  const int t = threadIdx.y * 32 + threadIdx.x;
#pragma unroll
  for (int half = 0; half < (GATED ? 2 : 1); ++half) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VEC; ++i) sums[threadIdx.y][threadIdx.x * VEC + i] = half ? s1[i] : s0[i];
    __syncthreads();
    const long long c = static_cast<long long>(blockIdx.x) * 32 * VEC + t;
    if (t < 32 * VEC && c < n) {
      float v = 0.0f;
#pragma unroll
      for (int y = 0; y < kDzRows; ++y) v += sums[y][t];
      row[half * n + c] = v;
    }
  }
}

__global__ void __launch_bounds__(256)
bias_sum_kernel(const float* __restrict__ partial, uint16_t* __restrict__ db, long long wide, long long total, int chunks,
                int f16) {
  grid_dependency_wait();
  grid_launch_dependents();
  const long long t = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (t >= total) return;
  const long long g = t / wide, c = t - g * wide;
  const float* src = partial + g * chunks * wide + c;
  float v = 0.0f;
  for (int i = 0; i < chunks; ++i) v += src[static_cast<long long>(i) * wide];
  db[t] = to16(v, f16 != 0);
}

// x of a gathered product by place, for the weight gradient, whose reduction runs over places: a copy of whole rows
// (16-byte words where a row allows it), bound by its bytes.  Fetching the rows by number inside the product costs the
// copies of a stage four times their time (2000 tokens x 2, 16 experts, 1024 x 2800: dW 129 us against 79 with this copy,
// which is 6 us of it).
template <int VEC>
__global__ void __launch_bounds__(256)
expert_rows_kernel(const uint16_t* __restrict__ x, const int* __restrict__ offsets, const int* __restrict__ order,
                   uint16_t* __restrict__ sorted, long long rows, long long src_rows, int div, long long k, int groups) {
  grid_dependency_wait();
  grid_launch_dependents();
  const long long place = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (place >= rows || place >= offsets[groups]) return;
  // a place of an expert's run that names no row is a row of zeros, as in the forward product (gathered_row)
  const int o = order[place];
  const long long row = o < 0 ? src_rows : o / div;
  const bool there = row < src_rows;
  const uint16_t* src = x + row * k;
  uint16_t* dst = sorted + place * k;
  for (long long c = static_cast<long long>(threadIdx.x & 31) * VEC; c < k; c += 32 * VEC) {
    if constexpr (VEC == 8) *reinterpret_cast<uint4*>(dst + c) = there ? *reinterpret_cast<const uint4*>(src + c) : make_uint4(0, 0, 0, 0);
    else dst[c] = there ? src[c] : static_cast<uint16_t>(0);
  }
}

// Row chunks of one group: enough blocks to fill the GPU on a long batch, at least 32 rows each on a short one.
static int dz_chunks(int64_t rows, int64_t groups) {
  const int64_t per = ceil_div64(rows, groups);
  int64_t c = ceil_div64(per, 32);
  const int64_t most = groups > 1 ? 16 : 64;
  return static_cast<int>(c < 1 ? 1 : c > most ? most : c);
}

static int64_t dz_pitch(int64_t wide) { return (wide + 7) / 8 * 8; }

static int64_t pad256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// Workspace: dz, then the partial sums of db, then (products over experts) x by place.
static size_t backward_workspace(int64_t rows, int64_t groups, int64_t n, int gated, int64_t sorted_k) {
  const int64_t wide = gated ? 2 * n : n;
  return static_cast<size_t>(pad256(rows * dz_pitch(wide) * 2) + pad256(groups * dz_chunks(rows, groups) * wide * 4) + rows * sorted_k * 2);
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static int run_product(const LinArgs& p, const ftb_config* cfg, int* status, cudaStream_t stream) {
  const int rc = launch_linear_umma(p, cfg, status, stream);
  return rc == FTB_E_UNSUPPORTED ? launch_linear_simt(p, stream) : rc;
}

constexpr int64_t kMaxExtent = 1ll << 30;

static int check_common(int dtype, int64_t rows, int64_t n, int64_t k, int activation, int gated) {
  if (dtype != FTB_BF16 && dtype != FTB_F16) return FTB_E_BAD_ARG;
  if (rows < 0 || n <= 0 || k <= 0) return FTB_E_BAD_ARG;
  if (activation < FTB_ACT_NONE || activation > FTB_ACT_SILU || gated < 0 || gated > 1) return FTB_E_BAD_ARG;
  if (rows > kMaxExtent || n > kMaxExtent / 2 || k > kMaxExtent) return FTB_E_TOO_LARGE;
  return FTB_OK;
}

// Knobs of ftb_linear and ftb_expert_linear, checked on every path, the CUDA-core one too.
static int check_config(const ftb_config* c, bool grouped) {
  if (!c) return FTB_OK;
  const int t = c->tile_n, s = c->split_k;
  if (t != 0 && t != 16 && t != 32 && t != 64 && t != 128 && t != 256) return FTB_E_BAD_CONFIG;
  if (c->cluster < 0 || c->cluster > 2 || c->stages < 0 || c->stages == 1 || c->stages > 8) return FTB_E_BAD_CONFIG;
  if (t == 256 && c->cluster == 1) return FTB_E_BAD_CONFIG;
  if (c->cluster == 2 && t != 0 && t < 128) return FTB_E_BAD_CONFIG;
  if (s != 0 && s != 1 && s != 2 && s != 4 && s != 8) return FTB_E_BAD_CONFIG;
  if (s > 1 && (grouped || c->cluster == 2 || t > 64)) return FTB_E_BAD_CONFIG;
  return FTB_OK;
}

// The three gradients of a product with an epilogue, dense (offsets null) or grouped.
static int backward_generic(int dtype, const void* x, const void* w, const int* offsets, const int* order, const void* dy,
                            const void* preact, void* dx, void* dw, void* db, int64_t rows, int64_t src_rows,
                            int64_t groups, int64_t n, int64_t k, int activation, int gated, int gather_div,
                            void* workspace, size_t workspace_bytes, int* status, cudaStream_t stream) {
  const int64_t wide = gated ? 2 * n : n;
  const bool need_z = gated || activation != FTB_ACT_NONE;
  if (rows > 0 && (!dy || (need_z && !preact) || (dx && !w) || (dw && !x))) return FTB_E_BAD_ARG;
  // dy itself serves as dz when nothing is applied to it and TMA can read its rows
  const bool own_dz = need_z || wide % 8 != 0 || !aligned16(dy);
  if (workspace_bytes < backward_workspace(rows, groups, n, gated, offsets ? k : 0) || !aligned16(workspace) ||
      (!workspace && workspace_bytes > 0))
    return FTB_E_WORKSPACE;
  const int rc = device_ok();
  if (rc) return rc;
  const int64_t ldz = own_dz ? dz_pitch(wide) : wide;
  uint16_t* dz = static_cast<uint16_t*>(workspace);
  const int64_t dz_bytes = pad256(rows * dz_pitch(wide) * 2);
  float* partial = db ? reinterpret_cast<float*>(static_cast<char*>(workspace) + dz_bytes) : nullptr;
  const bool write_dz = own_dz && (dx || dw) && rows > 0;
  const int f16 = dtype == FTB_F16;
  if (write_dz || db) {
    const int chunks = dz_chunks(rows, groups);
    const bool vec = n % 8 == 0 && aligned16(dy) && (!need_z || aligned16(preact));
    const int64_t gx = ceil_div64(n, vec ? 256 : 32);
    if (gx > 0x7fffffff) return FTB_E_TOO_LARGE;
    const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(chunks), static_cast<unsigned>(groups));
    const uint16_t* z = need_z ? static_cast<const uint16_t*>(preact) : nullptr;
    const uint16_t* d = static_cast<const uint16_t*>(dy);
    auto kern = vec ? (gated ? linear_dz_kernel<8, true> : linear_dz_kernel<8, false>)
                    : (gated ? linear_dz_kernel<1, true> : linear_dz_kernel<1, false>);
    int e = launch_overlapped(kern, grid, dim3(32, kDzRows), 0, 1, stream, d, z, write_dz ? dz : nullptr, ldz, partial, offsets,
                              rows, n, activation, f16, chunks);
    if (e) return e;
    if (db) {
      const int64_t total = groups * wide;
      e = launch_overlapped(bias_sum_kernel, dim3(static_cast<unsigned>(ceil_div64(total, 256))), dim3(256), 0, 1, stream,
                            partial, static_cast<uint16_t*>(db), wide, total, chunks, f16);
      if (e) return e;
    }
  }
  const uint16_t* g = own_dz ? dz : static_cast<const uint16_t*>(dy);
  if (dx && rows > 0) {
    LinArgs p;
    memset(&p, 0, sizeof(p));
    p.mode = offsets ? LIN_ROWS : LIN_DENSE;
    p.f16 = f16;
    p.a = static_cast<const uint16_t*>(w);
    p.lda = k;
    p.a_gs = wide * k;
    p.a_mn = 1;
    p.b = g;
    p.ldb = ldz;
    p.I = k;
    p.J = rows;
    p.K = wide;
    p.groups = static_cast<int>(groups);
    p.offsets = offsets;
    p.rows = rows;
    p.src_rows = rows;
    p.out = static_cast<uint16_t*>(dx);
    p.ldo = k;
    const int e = run_product(p, nullptr, status, stream);
    if (e) return e;
  }
  if (dw) {
    if (rows == 0) return launch_status(cudaMemsetAsync(dw, 0, static_cast<size_t>(groups) * wide * k * 2, stream));
    if (gather_div) {
      uint16_t* sorted = reinterpret_cast<uint16_t*>(static_cast<char*>(workspace) + dz_bytes + pad256(groups * dz_chunks(rows, groups) * wide * 4));
      const bool vec = k % 8 == 0 && aligned16(x);
      const int e = launch_overlapped(vec ? expert_rows_kernel<8> : expert_rows_kernel<1>,
                                      dim3(static_cast<unsigned>(ceil_div64(rows, 8))), dim3(256), 0, 1, stream,
                                      static_cast<const uint16_t*>(x), offsets, order, sorted, rows, src_rows, gather_div, k,
                                      static_cast<int>(groups));
      if (e) return e;
      x = sorted;
    }
    LinArgs p;
    memset(&p, 0, sizeof(p));
    p.mode = offsets ? LIN_REDUCE : LIN_DENSE;
    p.f16 = f16;
    p.a = static_cast<const uint16_t*>(x);
    p.lda = k;
    p.a_mn = 1;
    p.b = g;
    p.ldb = ldz;
    p.b_mn = 1;
    p.I = k;
    p.J = wide;
    p.K = rows;
    p.groups = static_cast<int>(groups);
    p.offsets = offsets;
    p.rows = rows;
    p.src_rows = rows;
    p.out = static_cast<uint16_t*>(dw);
    p.ldo = k;
    p.out_gs = wide * k;
    return run_product(p, nullptr, status, stream);
  }
  return FTB_OK;
}

}  // namespace ftb

extern "C" {

int ftb_linear(int dtype, const void* x, const void* w, const void* bias, const void* residual, void* out, void* preact,
               int64_t tokens, int64_t n, int64_t k, int activation, int gated, const ftb_config* cfg, int* status,
               void* stream) {
  using namespace ftb;
  int rc = check_common(dtype, tokens, n, k, activation, gated);
  if (!rc) rc = check_config(cfg, false);
  if (rc) return rc;
  if (tokens == 0) return FTB_OK;
  if (!x || !w || !out) return FTB_E_BAD_ARG;
  rc = device_ok();
  if (rc) return rc;
  LinArgs p;
  memset(&p, 0, sizeof(p));
  p.mode = LIN_DENSE;
  p.f16 = dtype == FTB_F16;
  p.a = static_cast<const uint16_t*>(w);
  p.lda = k;
  p.b = static_cast<const uint16_t*>(x);
  p.ldb = k;
  p.I = n;
  p.J = tokens;
  p.K = k;
  p.groups = 1;
  p.rows = tokens;
  p.bias = static_cast<const uint16_t*>(bias);
  p.residual = static_cast<const uint16_t*>(residual);
  p.out = static_cast<uint16_t*>(out);
  p.ldo = n;
  p.preact = static_cast<uint16_t*>(preact);
  p.ldp = gated ? 2 * n : n;
  p.act = activation;
  p.gated = gated;
  return run_product(p, cfg, status, static_cast<cudaStream_t>(stream));
}

size_t ftb_linear_backward_workspace_bytes(int64_t tokens, int64_t n, int64_t k, int gated) {
  if (ftb::check_common(FTB_BF16, tokens, n, k, 0, gated)) return 0;
  return ftb::backward_workspace(tokens, 1, n, gated, 0);
}

int ftb_linear_backward(int dtype, const void* x, const void* w, const void* dy, const void* preact, void* dx, void* dw,
                        void* db, int64_t tokens, int64_t n, int64_t k, int activation, int gated, void* workspace,
                        size_t workspace_bytes, int* status, void* stream) {
  using namespace ftb;
  const int rc = check_common(dtype, tokens, n, k, activation, gated);
  if (rc) return rc;
  if (!dx && !dw && !db) return tokens == 0 ? FTB_OK : FTB_E_BAD_ARG;  // (an empty dx has no address)
  return backward_generic(dtype, x, w, nullptr, nullptr, dy, preact, dx, dw, db, tokens, tokens, 1, n, k, activation,
                          gated, 0, workspace, workspace_bytes, status, static_cast<cudaStream_t>(stream));
}

static int check_experts(int64_t rows, int64_t top_k, int64_t experts) {
  if (experts <= 0 || top_k <= 0 || rows % top_k != 0) return FTB_E_BAD_ARG;
  if (experts > FTB_MAX_EXPERTS || top_k > FTB_MAX_TOP_K) return FTB_E_TOO_LARGE;
  return FTB_OK;
}

int ftb_expert_linear(int dtype, const void* x, const void* w, const void* bias, const int32_t* offsets,
                      const int32_t* order, void* out, void* preact, int64_t rows, int64_t top_k, int64_t experts,
                      int64_t n, int64_t k, int activation, int gated, int gather, const ftb_config* cfg, int* status,
                      void* stream) {
  using namespace ftb;
  int rc = check_common(dtype, rows, n, k, activation, gated);
  if (!rc) rc = check_experts(rows, top_k, experts);
  if (!rc) rc = check_config(cfg, true);
  if (rc) return rc;
  if (gather < 0 || gather > 1) return FTB_E_BAD_ARG;
  if (rows == 0) return FTB_OK;
  if (!x || !w || !out || !offsets || (gather && !order)) return FTB_E_BAD_ARG;
  rc = device_ok();
  if (rc) return rc;
  const int64_t wide = gated ? 2 * n : n;
  LinArgs p;
  memset(&p, 0, sizeof(p));
  p.mode = LIN_ROWS;
  p.f16 = dtype == FTB_F16;
  p.a = static_cast<const uint16_t*>(w);
  p.lda = k;
  p.a_gs = wide * k;
  p.b = static_cast<const uint16_t*>(x);
  p.ldb = k;
  p.I = n;
  p.J = rows;
  p.K = k;
  p.groups = static_cast<int>(experts);
  p.offsets = offsets;
  p.order = order;
  p.gather_div = gather ? static_cast<int>(top_k) : 0;
  p.rows = rows;
  p.src_rows = gather ? rows / top_k : rows;
  p.bias = static_cast<const uint16_t*>(bias);
  p.bias_gs = wide;
  p.out = static_cast<uint16_t*>(out);
  p.ldo = n;
  p.preact = static_cast<uint16_t*>(preact);
  p.ldp = wide;
  p.act = activation;
  p.gated = gated;
  return run_product(p, cfg, status, static_cast<cudaStream_t>(stream));
}

size_t ftb_expert_linear_backward_workspace_bytes(int64_t rows, int64_t experts, int64_t n, int64_t k, int gated) {
  if (ftb::check_common(FTB_BF16, rows, n, k, 0, gated) || check_experts(rows, 1, experts)) return 0;
  return ftb::backward_workspace(rows, experts, n, gated, k);
}

int ftb_expert_linear_backward(int dtype, const void* x, const void* w, const int32_t* offsets, const int32_t* order,
                               const void* dy, const void* preact, void* dx, void* dw, void* db, int64_t rows,
                               int64_t top_k, int64_t experts, int64_t n, int64_t k, int activation, int gated, int gather,
                               void* workspace, size_t workspace_bytes, int* status, void* stream) {
  using namespace ftb;
  int rc = check_common(dtype, rows, n, k, activation, gated);
  if (!rc) rc = check_experts(rows, top_k, experts);
  if (rc) return rc;
  if (gather < 0 || gather > 1 || !offsets || (rows > 0 && gather && !order)) return FTB_E_BAD_ARG;
  if (!dx && !dw && !db) return rows == 0 ? FTB_OK : FTB_E_BAD_ARG;
  return backward_generic(dtype, x, w, offsets, order, dy, preact, dx, dw, db, rows, gather ? rows / top_k : rows, experts,
                          n, k, activation, gated, gather ? static_cast<int>(top_k) : 0, workspace, workspace_bytes,
                          status, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
