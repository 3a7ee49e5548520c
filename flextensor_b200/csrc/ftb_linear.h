// One product with an epilogue, as the launchers describe it to the kernels that can run it.
#pragma once
#include "ftb_lm.cuh"

namespace ftb {

// Every product of the feed-forward operators has the same shape:
//   out[j, i] = epilogue( sum over k of A[i, k] * B[j, k] ),   i contiguous in `out`,
// with features on i and tokens (or, for a weight's gradient, the weight's rows) on j.
enum { LIN_DENSE = 0,   // one product
       LIN_ROWS = 1,    // j are sorted places, split by `offsets` into groups; A of group g
       LIN_REDUCE = 2 }; // k are sorted places, split by `offsets`, of operands sorted already; one result per group

struct LinArgs {
  int mode, f16;
  // a_mn = 0: A[i][k], k contiguous; 1: A[k][i], i contiguous.  Strides in elements.  The same for B.
  const uint16_t* a;
  long long lda, a_gs;
  int a_mn;
  const uint16_t* b;
  long long ldb;
  int b_mn;
  long long I, J, K;  // gated: A has 2 I rows, gate rows first
  int groups;
  const int* offsets;   // [groups + 1], or null for LIN_DENSE
  const int* order;     // sorted place -> row * gather_div + slot
  int gather_div;       // 0: the operand indexed by sorted places is sorted already; else it is gathered
  long long rows;       // sorted places (capacity); offsets are clamped to it
  long long src_rows;   // rows of the gathered operand
  const uint16_t* bias;
  long long bias_gs;
  const uint16_t* residual;  // pitch ldo
  uint16_t* out;
  long long ldo, out_gs;
  uint16_t* preact;
  long long ldp;
  int act, gated;
};

// Places [lo, hi) of group g.  Offsets come from device memory: whatever they hold, no access leaves the tensors.
__device__ __forceinline__ void group_range(const int* offsets, int g, long long rows, int* lo, int* hi) {
  const int cap = static_cast<int>(rows);
  const int a = offsets[g], b = offsets[g + 1];
  *lo = min(max(a, 0), cap);
  *hi = min(max(b, *lo), cap);
}

// Row of the gathered operand behind sorted place p, or -1.
__device__ __forceinline__ long long gathered_row(const LinArgs& p, long long place) {
  if (p.gather_div == 0) return place;
  const int o = p.order[place];
  if (o < 0) return -1;
  const long long r = o / p.gather_div;
  return r < p.src_rows ? r : -1;
}

int launch_linear_simt(const LinArgs& p, cudaStream_t stream);
// tcgen05 kernel; FTB_E_UNSUPPORTED when TMA cannot address an operand.
int launch_linear_umma(const LinArgs& p, const ftb_config* cfg, int* status, cudaStream_t stream);

}  // namespace ftb
