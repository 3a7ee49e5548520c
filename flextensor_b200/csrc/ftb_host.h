// Host-side helpers shared by the translation units of the library.
#pragma once
#include "../../include/ftb200.h"
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

namespace ftb {

void set_last_cuda_error(int code);
void count_launch();
// FTB_OK when the current device is compute capability 10.x.
int device_ok();
// SM count of the current device (cached per device).
int sm_count();
// Device address of the library's own status word, used when the caller passes none.
int* fallback_status();

// Shared memory that a CTA of a pair (cta_group::2) asks for.  A pair takes tensor memory on both of its SMs before its
// CTAs meet at a cluster barrier, and nothing says that the two are taken at once: two pairs on the same two SMs, of one
// kernel or of any two on different streams, could each hold the columns that the other waits for.  So every pair asks
// for more than half of an SM's shared memory, and no SM ever holds CTAs of two pairs.  (Single CTAs and split clusters may
// stand beside a pair: they hold tensor memory without waiting for another CTA, and give it back.)
constexpr size_t kSmSharedBytes = 228 * 1024;  // of an SM, of which the system keeps 1 KB per resident CTA
constexpr size_t kCtaReserved = 1024;
constexpr size_t kPairSharedFloor = 114 * 1024;
static_assert(2 * (kPairSharedFloor + kCtaReserved) > kSmSharedBytes, "two CTAs of pairs must not fit an SM");
inline size_t pair_shared_bytes(size_t need) { return need < kPairSharedFloor ? kPairSharedFloor : need; }

// Options of gemm_generic beyond the plain (batched) product.
struct GemmExtras {
  int a_broadcast;        // 1: every batch entry multiplies the same A (A holds one matrix)
  const float* row_bias;  // fp32 output only: bias[i] added to row i of every result, may be null
};

// `extra_dst`: further buffers (num_extra of them) that receive the same result as `c`.
int gemm_generic(int kind, int out, const void* a, const void* b, void* c, int64_t batch, int64_t m,
                 int64_t n, int64_t k, int trans_a, int trans_b, const ftb_config* user, int* status,
                 void* stream, void* const* extra_dst, int num_extra, const GemmExtras* extras = nullptr);

// CUDA-core GEMM for operands whose pitches or bases break the 16-byte rules of TMA.
int simt_gemm(int kind, int out, const void* a, const void* b, void* c, int64_t batch, int64_t m, int64_t n,
              int64_t k, int trans_a, int trans_b, void* stream);

int conv2d_generic(const float* in, const float* weight, const float* bias, float* out, int64_t n,
                   int64_t c, int64_t h, int64_t w, int64_t k, int64_t r, int64_t s, int stride_h,
                   int stride_w, int pad_h, int pad_w, int dil_h, int dil_w, int groups,
                   const ftb_config* user, void* workspace, size_t workspace_bytes, int* status,
                   void* stream, float* const* extra_dst = nullptr, int num_extra = 0, int filter_mode = 0,
                   int layout = 0);

}  // namespace ftb
