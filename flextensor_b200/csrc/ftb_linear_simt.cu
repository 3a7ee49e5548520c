// CUDA-core form of the products with an epilogue: the path of operands that TMA cannot address (a row pitch or a base
// that is no multiple of 16 bytes).  64 x 64 results per CTA, 4 x 4 per thread, fp32 accumulation in ascending k,
// every access bounds-checked.  A correctness path like ftb_simt_gemm.cu: bound by its shared-memory reads (two words
// per two multiply-adds), an order of magnitude behind the tcgen05 kernel.
#include "ftb_linear.h"

namespace ftb {

template <bool GATED>
__global__ void __launch_bounds__(256) linear_simt_kernel(const LinArgs p) {
  constexpr int T = 64, TK = 16, SUBS = GATED ? 2 : 1;
  __shared__ float As[SUBS][TK][T + 1];
  __shared__ float Bs[TK][T + 1];
  grid_dependency_wait();
  grid_launch_dependents();
  const bool f16 = p.f16 != 0;
  const int g = blockIdx.z;
  int lo = 0, hi = 0;
  if (p.mode != LIN_DENSE) group_range(p.offsets, g, p.rows, &lo, &hi);
  const long long K = p.mode == LIN_REDUCE ? hi - lo : p.K;
  const long long J = p.mode == LIN_ROWS ? hi - lo : p.J;
  const uint16_t* a = p.a + g * p.a_gs;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const long long i0 = static_cast<long long>(blockIdx.x) * T;

  for (long long j0 = static_cast<long long>(blockIdx.y) * T; j0 < J; j0 += static_cast<long long>(gridDim.y) * T) {
    float acc[SUBS][4][4] = {};
    for (long long k0 = 0; k0 < K; k0 += TK) {
      for (int e = threadIdx.x; e < T * TK; e += 256) {
        // the contiguous dimension runs over neighbouring threads
        const int ai = p.a_mn ? e % T : e / TK, ak = p.a_mn ? e / T : e % TK;
        const long long i = i0 + ai, k = k0 + ak;
#pragma unroll
        for (int s = 0; s < SUBS; ++s) {
          float v = 0.0f;
          if (i < p.I && k < K) {
            const long long row = i + (s ? p.I : 0);
            if (p.mode == LIN_REDUCE) {
              v = from16(a[(lo + k) * p.lda + row], f16);
            } else {
              v = from16(p.a_mn ? a[k * p.lda + row] : a[row * p.lda + k], f16);
            }
          }
          As[s][ak][ai] = v;
        }
        const int bj = p.b_mn ? e % T : e / TK, bk = p.b_mn ? e / T : e % TK;
        const long long j = j0 + bj, kb = k0 + bk;
        float v = 0.0f;
        if (j < J && kb < K) {
          if (p.mode == LIN_REDUCE) {
            v = from16(p.b[(lo + kb) * p.ldb + j], f16);
          } else if (p.mode == LIN_ROWS) {
            const long long r = gathered_row(p, lo + j);
            if (r >= 0) v = from16(p.b[r * p.ldb + kb], f16);
          } else {
            v = from16(p.b_mn ? p.b[kb * p.ldb + j] : p.b[j * p.ldb + kb], f16);
          }
        }
        Bs[bk][bj] = v;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < TK; ++k) {
        float bv[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) bv[c] = Bs[k][ty * 4 + c];
#pragma unroll
        for (int s = 0; s < SUBS; ++s)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float av = As[s][k][tx + 16 * r];
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[s][r][c] = fmaf(av, bv[c], acc[s][r][c]);
          }
      }
      __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const long long i = i0 + tx + 16 * r;
      if (i >= p.I) continue;
      float b0 = 0.0f, b1 = 0.0f;
      if (p.bias) {
        b0 = from16(p.bias[g * p.bias_gs + i], f16);
        if (GATED) b1 = from16(p.bias[g * p.bias_gs + p.I + i], f16);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const long long j = j0 + ty * 4 + c;
        if (j >= J) continue;
        const long long row = p.mode == LIN_ROWS ? lo + j : j;
        const float z = acc[0][r][c] + b0;
        float v = act_value(z, p.act);
        if (p.preact) p.preact[row * p.ldp + i] = to16(z, f16);
        if (GATED) {
          const float u = acc[SUBS - 1][r][c] + b1;
          if (p.preact) p.preact[row * p.ldp + p.I + i] = to16(u, f16);
          v *= u;
        }
        const long long at = g * p.out_gs + row * p.ldo + i;
        if (p.residual) v += from16(p.residual[at], f16);
        p.out[at] = to16(v, f16);
      }
    }
  }
}

int launch_linear_simt(const LinArgs& p, cudaStream_t stream) {
  const int64_t most_j = p.mode == LIN_ROWS ? p.rows : p.J;
  int64_t gy = ceil_div64(most_j, 64);
  // rows spread over the groups: about twice the average group's tiles, the kernel walks what is left
  if (p.mode == LIN_ROWS) gy = ceil_div64(2 * most_j, 64 * static_cast<int64_t>(p.groups));
  if (gy < 1) gy = 1;
  if (gy > 65535) gy = 65535;
  const int64_t gx = ceil_div64(p.I, 64);
  if (gx > 0x7fffffff) return FTB_E_TOO_LARGE;
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy), static_cast<unsigned>(p.groups));
  return launch_overlapped(p.gated ? linear_simt_kernel<true> : linear_simt_kernel<false>, grid, dim3(256), 0, 1, stream, p);
}

}  // namespace ftb
