// The products with an epilogue on tcgen05: out[j, i] = epilogue(sum over k of A[i, k] B[j, k]).
//
// Features (i) lie on the 128 lanes of tensor memory and tokens (j) on its columns, in every direction: a tile of few
// tokens is then a narrow accumulator (16 columns for one token) instead of 128 mostly empty rows, a thread of the
// epilogue owns one feature, so its bias is one register, and 32 lanes store 32 neighbouring features of a token.
//
//   warp 0      producer: TMA tiles of A and B into 128-byte swizzled stages of 64 k; rows named by a list (tokens of
//               an expert, or the reduction of its weight gradient) come by gather4, four rows per lane and copy, and a
//               row past the end of its expert is asked for outside the tensor, which fills it with zeros
//   warp 1, 2   issuers of tcgen05.mma, one per A sub-tile.  The whole warp runs the loop and one elected lane issues:
//               addresses and descriptors then stay in uniform registers.  Run by a single lane, a stage of four MMAs
//               took about 900 cycles whatever its tile, now 500 in a pair and 420 alone (256 x 4096 x 4096: 31.4 -> 20.9 us
//               when it was changed; 23.3 as it stands)
//   warp 3      second loader where rows are fetched by number (a gather4 costs its loader about 50 ns)
//   warps 4..   epilogue: tcgen05.ld -> bias, activation, gate, residual -> stores
//
// Forms: FORM_PLAIN one A sub-tile; FORM_GATED two, the gate rows and the others of the same features, whose
// accumulators share lanes and columns, so the gate is applied in registers; FORM_WIDE two neighbouring feature tiles
// over the same tokens (a byte of B feeds twice the math).  PAIR runs two CTAs as one cta_group::2 unit.
// SPLIT gives the reduction of one tile to the CTAs of a cluster.  Every CTA finishes a run of the tile's columns; the
// others write their fp32 partial sums of those into its shared memory, where they are added in rank order after one
// cluster barrier (pulling them after the barrier instead cost 1.5 us more, and a second barrier before the exit).
//
// Waits are bounded as in ftb_umma_kernel.cuh: a role that gives up sets a status bit and the CTA leaves through its
// normal teardown.
//
// What bounds it, measured on a B200 (bf16, device time in a CUDA graph of calls on rotating operands larger than L2, after
// 0.4 s of the same load, so under the power cap where it applies; in brackets the first milliseconds):
//   4096 x 4096 x 4096            114 us  1.20 PFLOP/s at 1485 MHz, 0.86 of the sustained matrix rate (97 us, 1.41, 0.87 of
//                                         the burst rate); rows through the SM's port (256 a stage for 512 cycles of math)
//   8192 x (2 x 8192) x 4096 gated 862 us 1.28 PFLOP/s at 1425 MHz, 0.91 of the sustained rate (809 us): the power cap
//   1 x 4096 x 4096               9.7 us  3.4 TB/s: 5.1 us of reading W, then launch, first copies and the exchange of the
//                                         partial sums; four CTAs per tile (eight: 11.7, two: 13.6, one: 21.4)
//   48 x (2 x 8192) x 2048 gated  16.9 us 4.0 TB/s: 10.4 us of reading W
//   1237 x 2048 x 1000            10.6 us, with GELU, bias, residual and preact 15.6: one wave of tiles whose epilogue
//                                         nothing covers; 2051 columns, stored in 2-byte accesses: 16.2
//   15360 places of 32 experts x 2048 x 2048  156 us  0.82 PFLOP/s of useful work (132 us, 0.98): a quarter of the tiles' rows
//                                         are the ends of groups; the same rows gathered by number 186 us (12 cycles a row)
#include "ftb_linear.h"
#include "ftb_ptx.cuh"
#include "ftb_tmap.h"

#include <mutex>

namespace ftb {

enum { FORM_PLAIN = 0, FORM_GATED = 1, FORM_WIDE = 2 };
constexpr int kLinStages = 8;
constexpr uint32_t kSubBytes = 128 * 128;  // 128 rows x 64 elements
constexpr int kKBlock = 64;

// Division by a number known on the host: the high word of a product with floor(2^32 / d) is at most one short.
struct FastDiv {
  uint32_t d, m;
};
static FastDiv fast_div(int64_t d) {
  FastDiv f;
  f.d = static_cast<uint32_t>(d);
  f.m = d > 1 ? static_cast<uint32_t>((1ull << 32) / static_cast<uint64_t>(d)) : 0xffffffffu;
  return f;
}
__device__ __forceinline__ uint32_t div_by(uint32_t x, const FastDiv& f, uint32_t* rest) {
  uint32_t q = __umulhi(x, f.m), r = x - q * f.d;
  if (r >= f.d) {
    ++q;
    r -= f.d;
  }
  *rest = r;
  return q;
}

struct LinUmma {
  LinArgs q;
  int bn, bj;            // tokens per tile, and of those staged per CTA
  int stages, split;
  int most_rows;         // LIN_ROWS: token tiles of a plan, at most (offsets that are none cannot ask for more)
  int tiles_i, tiles_j;  // tiles_j: LIN_DENSE and LIN_REDUCE
  int feat, sub_off;     // features per tile; feature rows between the A sub-tiles
  int band;              // token tiles walked together before the next feature tile
  FastDiv by_i, by_group, by_span, by_band, by_last;  // tiles_i, tiles_i tiles_j, a band's tiles, its width, the last's
  int acc_slots;         // accumulators in turn (FORM_WIDE: one per sub-tile)
  uint32_t tmem_cols;
  uint32_t idesc;
  uint32_t a_lbo, b_lbo, a_kadv, b_kadv;
  int oob_b;             // a row past the tensors whose rows are fetched by number
  int vec;               // rows of out, residual and preact start on 16 bytes
  int* status;
};

// Tiled maps of the operands, and maps whose boxes are one row high for rows fetched by number.
struct LinMaps {
  CUtensorMap a, b;            // a stage's boxes
  CUtensorMap a_rows, b_rows;  // one row high, for rows fetched by number
  CUtensorMap a16, b16;        // 16 k high, for the last block of a reduction
};

struct LinTile {
  int g, ti, tj, lo, cnt;  // group, feature tile, token tile; the group's first place and number of places
};

__device__ __forceinline__ LinTile lin_tile(const LinUmma& p, const int* tstart, int t) {
  LinTile c;
  c.g = 0;
  c.lo = 0;
  c.cnt = 0;
  uint32_t r;
  if (p.q.mode == LIN_ROWS) {
    // feature tiles run fastest; then the group whose token tiles hold this one
    const int tok = static_cast<int>(div_by(t, p.by_i, &r));
    c.ti = static_cast<int>(r);
    int a = 0, b = p.q.groups;
    while (b - a > 1) {
      const int mid = (a + b) >> 1;
      if (tstart[mid] <= tok) a = mid;
      else b = mid;
    }
    c.g = a;
    c.tj = tok - tstart[a];
    int hi;
    group_range(p.q.offsets, a, p.q.rows, &c.lo, &hi);
    c.cnt = hi - c.lo;
    return c;
  }
  r = t;
  if (p.q.mode == LIN_REDUCE) {
    c.g = static_cast<int>(div_by(t, p.by_group, &r));
    int hi;
    group_range(p.q.offsets, c.g, p.q.rows, &c.lo, &hi);
    c.cnt = hi - c.lo;
  }
  // bands of `band` token tiles: inside one, token tiles run fastest
  uint32_t q, x;
  const int first = static_cast<int>(div_by(r, p.by_span, &q)) * p.band;
  c.ti = static_cast<int>(first + p.band <= p.tiles_j ? div_by(q, p.by_band, &x) : div_by(q, p.by_last, &x));
  c.tj = first + static_cast<int>(x);
  return c;
}

// Columns of a tile that one CTA of a split reduction finishes: a multiple of four.
__host__ __device__ __forceinline__ int split_share(int columns, int split) { return ((columns + split - 1) / split + 3) & ~3; }

__device__ __forceinline__ int lin_blocks(const LinUmma& p, const LinTile& c) {
  return p.q.mode == LIN_REDUCE ? (c.cnt + kKBlock - 1) / kKBlock : static_cast<int>((p.q.K + kKBlock - 1) / kKBlock);
}

// The activation on NC values: one branch, then straight-line code.
template <int NC>
__device__ __forceinline__ void act_values(float (&v)[NC], int act) {
  if (act == FTB_ACT_SILU) {
#pragma unroll
    for (int c = 0; c < NC; ++c) v[c] = act_value(v[c], FTB_ACT_SILU);
  } else if (act == FTB_ACT_GELU) {
#pragma unroll
    for (int c = 0; c < NC; ++c) v[c] = act_value(v[c], FTB_ACT_GELU);
  } else if (act == FTB_ACT_GELU_TANH) {
#pragma unroll
    for (int c = 0; c < NC; ++c) v[c] = act_value(v[c], FTB_ACT_GELU_TANH);
  } else if (act == FTB_ACT_RELU) {
#pragma unroll
    for (int c = 0; c < NC; ++c) v[c] = act_value(v[c], FTB_ACT_RELU);
  }
}

// The epilogue of 16 columns (tokens) by one warp, whose lanes hold 32 neighbouring features.  The arithmetic runs as
// the accumulator lies, a feature per lane.  Where every row of the results starts on 16 bytes (`vec`) a warp then turns
// its 16 x 32 values round through 2.25 KB of shared memory and a lane loads and stores eight features of a token at a
// time.  Rows of other pitches keep 2-byte accesses, 64 contiguous bytes per warp, without predicates where all columns
// are tokens (GELU with bias, residual and preact, 1237 x 2048 x 1000: 15.6 us; 2051 columns: 16.2, with predicates 21.2).
constexpr int kCols = 16;          // columns a thread holds at a time
constexpr int kTurnPitch = 36;     // floats between two tokens: a lane's 16-byte reads meet no bank twice
constexpr int kTurnFloats = kCols * kTurnPitch;

struct WarpCols {
  float* turn;        // this warp's staging
  int lane;
  bool live;          // the lane's feature exists
  bool live8;         // so do the eight features that the lane moves in the turned layout
  int valid;          // columns that are tokens of this tile
};

// Reads the residual before the sums are ready: turned, 2 x 8 features; else 16 tokens of the lane's feature.  `r` is
// the lane's own element of column 0.
__device__ __forceinline__ void lin_residual(bool vec, const WarpCols& w, uint32_t (&res)[kCols], const uint16_t* r,
                                             long long pitch) {
  if (vec) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (w.live8 && (w.lane >> 2) + 8 * h < w.valid) x = *reinterpret_cast<const uint4*>(r + (h ? 8 * pitch : 0));
      res[4 * h] = x.x;
      res[4 * h + 1] = x.y;
      res[4 * h + 2] = x.z;
      res[4 * h + 3] = x.w;
    }
  } else if (w.live && w.valid >= kCols) {
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      res[c] = *r;
      r += pitch;
    }
  } else {
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      res[c] = w.live && c < w.valid ? *r : 0u;
      r += pitch;
    }
  }
}

// Rounds and stores the warp's 16 x 32 values; `o` is the lane's own element of column 0, `res` null or the residual.
__device__ __forceinline__ void lin_store(bool vec, bool f16, const WarpCols& w, float (&v)[kCols], uint16_t* o,
                                          long long pitch, const uint32_t* res) {
  if (vec) {
    __syncwarp();
#pragma unroll
    for (int c = 0; c < kCols; ++c) w.turn[c * kTurnPitch + w.lane] = v[c];
    __syncwarp();
    const int tok = w.lane >> 2;
    const float4* from = reinterpret_cast<const float4*>(w.turn + tok * kTurnPitch + (w.lane & 3) * 8);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 a = from[h * 8 * kTurnPitch / 4], b = from[h * 8 * kTurnPitch / 4 + 1];
      float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      if (res) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 r = unpack16(res[4 * h + e], f16);
          x[2 * e] += r.x;
          x[2 * e + 1] += r.y;
        }
      }
      if (w.live8 && tok + 8 * h < w.valid)
        *reinterpret_cast<uint4*>(o + (h ? 8 * pitch : 0)) =
            make_uint4(pack16(x[0], x[1], f16), pack16(x[2], x[3], f16), pack16(x[4], x[5], f16), pack16(x[6], x[7], f16));
    }
  } else if (w.live) {
    float x[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c) x[c] = res ? v[c] + from16(static_cast<uint16_t>(res[c]), f16) : v[c];
    if (w.valid >= kCols) {
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        *o = to16(x[c], f16);
        o += pitch;
      }
    } else {
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        if (c < w.valid) *o = to16(x[c], f16);
        o += pitch;
      }
    }
  }
}

// RICH = false: nothing but the store.  (In one kernel with the rest, the jumps over its code cost a short reduction
// as much as the store itself: 600 cycles per 16 columns and warp.)
template <bool GATED, bool RICH>
__device__ __forceinline__ void lin_finish(const LinArgs& q, bool vec, const WarpCols& w, float (&v)[kCols],
                                           float (&u)[kCols], const uint32_t (&res)[kCols], float b0, float b1,
                                           uint16_t* out, uint16_t* preact) {
  const bool f16 = q.f16 != 0;
  if constexpr (!RICH) {
    lin_store(vec, f16, w, v, out, q.ldo, nullptr);
    return;
  }
  if (q.bias) {
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      v[c] += b0;
      if constexpr (GATED) u[c] += b1;
    }
  }
  if (q.preact) {
    lin_store(vec, f16, w, v, preact, q.ldp, nullptr);
    if constexpr (GATED) lin_store(vec, f16, w, u, preact + q.I, q.ldp, nullptr);
  }
  if (q.act) act_values<kCols>(v, q.act);
  if constexpr (GATED) {
#pragma unroll
    for (int c = 0; c < kCols; ++c) v[c] *= u[c];
  }
  lin_store(vec, f16, w, v, out, q.ldo, q.residual ? res : nullptr);
}

// The same for four tokens of one feature (after a split reduction).
template <bool GATED>
__device__ __forceinline__ void lin_finish4(const LinArgs& q, float (&v)[4], float (&u)[4], float b0, float b1,
                                            const uint16_t (&res)[4], long long i, long long row, int valid) {
  const bool f16 = q.f16 != 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] += b0;
    if constexpr (GATED) u[e] += b1;
  }
  if (q.preact) {
    uint16_t* z = q.preact + row * q.ldp + i;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < valid) {
        z[e * q.ldp] = to16(v[e], f16);
        if constexpr (GATED) z[e * q.ldp + q.I] = to16(u[e], f16);
      }
  }
  act_values<4>(v, q.act);
  uint16_t* out = q.out + row * q.ldo + i;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (GATED) v[e] *= u[e];
    if (q.residual) v[e] += from16(res[e], f16);
    if (e < valid) out[e * q.ldo] = to16(v[e], f16);
  }
}

template <bool PAIR, int FORM, int EPI, bool SPLIT, bool RICH>
__global__ void __launch_bounds__(128 + 32 * EPI, EPI == 4 ? 2 : 1)
linear_umma_kernel(const __grid_constant__ LinMaps maps, const __grid_constant__ LinUmma p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kLinStages];
  __shared__ __align__(8) uint64_t bar_empty[kLinStages];
  __shared__ __align__(8) uint64_t bar_tfull[2];
  __shared__ __align__(8) uint64_t bar_tempty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ int tstart[FTB_MAX_EXPERTS + 1];
  __shared__ int4 row_quads[2][16];  // rows of the copies that each loader warp issues
  constexpr int SUBS = FORM == FORM_PLAIN ? 1 : 2;
  static_assert(!SPLIT || (!PAIR && FORM != FORM_WIDE && EPI == 4), "the reduction is split in single-CTA tiles only");

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t b_bytes = static_cast<uint32_t>(p.bj) * 128u;
  const uint32_t stage_bytes = SUBS * kSubBytes + b_bytes;
  const uint32_t rank = (PAIR || SPLIT) ? cluster_ctarank() : 0u;
  const int unit = PAIR ? blockIdx.x >> 1 : SPLIT ? blockIdx.x / p.split : blockIdx.x;
  const int units = PAIR ? gridDim.x >> 1 : SPLIT ? gridDim.x / p.split : gridDim.x;
  const uint32_t stages = p.stages;
  const int mode = p.q.mode;

  if constexpr (SPLIT) cluster_arrive();  // this CTA runs: its shared memory can be written from now on
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (uint32_t s = 0; s < stages; ++s) {
      // Where the second loader has copies in some blocks only (the last of a reduction) it reports every block, so that
      // the ring never gets a turn ahead of it and its waits always mean the turn they ask about.
      mbar_init(smem_u32(&bar_full[s]), 1 + (mode == LIN_REDUCE ? (PAIR ? 2 : 1) : 0));
      mbar_init(smem_u32(&bar_empty[s]), SUBS);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&bar_tfull[a]), FORM == FORM_GATED ? 2 : 1);
      mbar_init(smem_u32(&bar_tempty[a]), (FORM == FORM_WIDE ? EPI / 2 : EPI) * (PAIR ? 2 : 1));
    }
    fence_mbar_init();
    fence_proxy_async_smem();
    prefetch_tmap(&maps.a);
    prefetch_tmap(mode == LIN_ROWS && p.q.gather_div != 0 ? &maps.b_rows : &maps.b);
  }
  // The kernel before this one may still run and may not hold all the tensor memory yet that it is going to need: this
  // one asks for its own only after it.
  grid_dependency_wait();
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(smem_u32(&tmem_slot), p.tmem_cols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(&tmem_slot), p.tmem_cols);
      tmem_relinquish();
    }
  }
  if (warp == 3 && mode == LIN_ROWS) {
    // token tiles before each group
    int base = 0;
    for (int g0 = 0; g0 < p.q.groups; g0 += 32) {
      int n = 0;
      if (g0 + lane < p.q.groups) {
        int lo, hi;
        group_range(p.q.offsets, g0 + lane, p.q.rows, &lo, &hi);
        n = (hi - lo + p.bn - 1) / p.bn;
      }
      int x = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      if (g0 + lane < p.q.groups) tstart[g0 + lane + 1] = min(base + x, p.most_rows);
      base = min(base + __shfl_sync(0xffffffffu, x, 31), p.most_rows);
    }
    if (lane == 0) tstart[0] = 0;
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();  // the peer's barriers exist before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_slot, 0);
  grid_launch_dependents();  // tensor memory is held: a successor's CTA on this SM cannot take it first

  const int total = mode == LIN_ROWS ? tstart[p.q.groups] * p.tiles_i : p.q.groups * p.tiles_i * p.tiles_j;
  const uint32_t full0 = smem_u32(&bar_full[0]), empty0 = smem_u32(&bar_empty[0]);
  const uint32_t tfull0 = smem_u32(&bar_tfull[0]), tempty0 = smem_u32(&bar_tempty[0]);
  const uint32_t slot_stride = FORM == FORM_WIDE ? static_cast<uint32_t>(p.bn) : static_cast<uint32_t>(p.bn) * SUBS;

  // Rows by number: tokens of a group (gather_j), or the places of a reduction's last block (gather_k), of which those
  // past the group are asked for outside the tensors.  Two warps share the copies.
  const bool gather_j = mode == LIN_ROWS && p.q.gather_div != 0;
  const bool gather_k = mode == LIN_REDUCE;
  if (warp == 0 || (warp == 3 && (gather_j || gather_k))) {
    // ------------------------------------------------------------ producer
    const int part = warp == 3 ? 1 : 0;
    const uint32_t tx = stage_bytes;
    const uint32_t sig0 = PAIR ? map_to_cta(full0, 0) : full0;
    int4* quads = row_quads[part];
    uint32_t s = 0, ph = 0, sa = smem_base;
    bool ok = true;
    for (int t = unit; t < total && ok; t += units) {
      const LinTile c = lin_tile(p, tstart, t);
      const int blocks = lin_blocks(p, c);
      const int per = SPLIT ? (blocks + p.split - 1) / p.split : blocks;
      const int kb0 = SPLIT ? static_cast<int>(rank) * per : 0, kb1 = min(blocks, kb0 + per);
      const int f0 = c.ti * p.feat + static_cast<int>(rank) * (PAIR ? 128 : 0);
      const int j0 = c.tj * p.bn + static_cast<int>(rank) * (PAIR ? p.bj : 0);
      const int half = p.bj >> 3;  // gather_j: quads of four rows per loader warp
      if (gather_j) {
        __syncwarp();
        if (lane < half) {
          int row[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = j0 + (part * half + lane) * 4 + e;
            const long long r = j < c.cnt ? gathered_row(p.q, c.lo + j) : -1;
            row[e] = r >= 0 ? static_cast<int>(r) : p.oob_b;
          }
          quads[lane] = make_int4(row[0], row[1], row[2], row[3]);
        }
        __syncwarp();
      }
      for (int kb = kb0; kb < kb1; ++kb) {
        const bool tail = gather_k && (kb + 1) * kKBlock > c.cnt;  // the block ends past the group
        // The last block of a group: whole runs of 16 places as tiles (an MMA takes 16), the places of the run in which
        // the group ends by number, those past it outside the tensors.
        const int runs = tail ? (c.cnt - kb * kKBlock) >> 4 : 0, odd = tail ? (c.cnt - kb * kKBlock) & 15 : 0;
        ok = __all_sync(0xffffffffu, mbar_wait(empty0 + 8 * s, ph ^ 1u, &abort_flag));
        if (!ok) {
          if (lane == 0) {
            atomicOr(p.status, FTB_DEV_WAIT_EMPTY);
            abort_flag = 1;
          }
          break;
        }
        if (elect_one()) {
          const uint32_t full = sig0 + 8 * s, sb = sa + SUBS * kSubBytes;
          const int kc = gather_k ? c.lo + kb * kKBlock : kb * kKBlock;
          if (part == 0) {
            const uint32_t bytes = tail ? tx / 4 * (runs + (odd ? 1 : 0)) : tx;
            if (!PAIR || rank == 0) mbar_expect_tx(full0 + 8 * s, PAIR ? 2 * bytes : bytes);
            if (!tail) {
#pragma unroll
              for (int sub = 0; sub < SUBS; ++sub) {
                const uint32_t dst = sa + sub * kSubBytes;
                const int f = f0 + sub * p.sub_off, g = gather_k ? 0 : c.g;
                if (p.q.a_mn) {
#pragma unroll
                  for (int b = 0; b < 2; ++b) {
                    if constexpr (PAIR) tma_load_3d_pair(dst + b * 8192u, &maps.a, full, f + b * 64, kc, g);
                    else tma_load_3d(dst + b * 8192u, &maps.a, full, f + b * 64, kc, g);
                  }
                } else {
                  if constexpr (PAIR) tma_load_3d_pair(dst, &maps.a, full, kc, f, g);
                  else tma_load_3d(dst, &maps.a, full, kc, f, g);
                }
              }
            }
            if (p.q.b_mn) {
              if (!tail) {
                for (int b = 0; b * 64 < p.bj; ++b) {
                  if constexpr (PAIR) tma_load_3d_pair(sb + b * 8192u, &maps.b, full, j0 + b * 64, kc, 0);
                  else tma_load_3d(sb + b * 8192u, &maps.b, full, j0 + b * 64, kc, 0);
                }
              }
            } else if (!gather_j) {
              if constexpr (PAIR) tma_load_3d_pair(sb, &maps.b, full, kc, c.lo + j0, 0);
              else tma_load_3d(sb, &maps.b, full, kc, c.lo + j0, 0);
            }
          }
          if (gather_j) {
            uint32_t dst = sb + part * half * 512u;
#pragma unroll 4
            for (int e = 0; e < half; ++e, dst += 512u) {
              const int4 r = quads[e];
              if constexpr (PAIR) tma_gather4_pair(dst, &maps.b_rows, full, kc, r.x, r.y, r.z, r.w);
              else tma_gather4(dst, &maps.b_rows, full, kc, r.x, r.y, r.z, r.w);
            }
          }
          if (tail) {
            for (int x = 0; x < 2 * SUBS + (p.bj >> 6); ++x) {
              const bool in_a = x < 2 * SUBS;
              const int y = x - 2 * SUBS;
              const uint32_t dst = in_a ? sa + x * 8192u : sb + y * 8192u;
              const int col = in_a ? f0 + (x >> 1) * p.sub_off + (x & 1) * 64 : j0 + y * 64;
              if ((x & 1) != part) continue;  // the two loader warps take turns
              const CUtensorMap* m16 = in_a ? &maps.a16 : &maps.b16;
              const CUtensorMap* m1 = in_a ? &maps.a_rows : &maps.b_rows;
              for (int r = 0; r < runs; ++r) {
                if constexpr (PAIR) tma_load_3d_pair(dst + r * 2048u, m16, full, col, kc + r * 16, 0);
                else tma_load_3d(dst + r * 2048u, m16, full, col, kc + r * 16, 0);
              }
              for (int e = 0; odd && e < 4; ++e) {
                const int k = e * 4, base = kc + runs * 16;
                const int r0 = k < odd ? base + k : p.oob_b, r1 = k + 1 < odd ? base + k + 1 : p.oob_b;
                const int r2 = k + 2 < odd ? base + k + 2 : p.oob_b, r3 = k + 3 < odd ? base + k + 3 : p.oob_b;
                const uint32_t at = dst + runs * 2048u + e * 512u;
                if constexpr (PAIR) tma_gather4_pair(at, m1, full, col, r0, r1, r2, r3);
                else tma_gather4(at, m1, full, col, r0, r1, r2, r3);
              }
            }
          }
          if (gather_k && part == 1) {
            if constexpr (PAIR) mbar_arrive_cluster(full);
            else mbar_arrive(full);
          }
        }
        __syncwarp();
        sa += stage_bytes;
        if (++s == stages) {
          s = 0;
          ph ^= 1u;
          sa = smem_base;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1 || (SUBS == 2 && warp == 2)) {
    // ------------------------------------------------------------ MMA issuers (leader CTA of a pair)
    const uint32_t sub = warp - 1;
    if (!PAIR || rank == 0) {
      const uint32_t idesc = p.idesc;
      const uint32_t a_hi = smem_desc_hi(p.a_lbo, 1024, 2), b_hi = smem_desc_hi(p.b_lbo, 1024, 2);
      const uint32_t a_lo0 = smem_desc_lo(smem_base + sub * kSubBytes, p.a_lbo);
      const uint32_t b_lo0 = smem_desc_lo(smem_base + SUBS * kSubBytes, p.b_lbo);
      const uint32_t a_k = p.a_kadv >> 4, b_k = p.b_kadv >> 4, stage_enc = stage_bytes >> 4;
      uint32_t s = 0, ph = 0, off = 0;
      bool ready = false;
      int local = 0;
      bool ok = true;
      for (int t = unit; t < total && ok; t += units, ++local) {
        const LinTile c = lin_tile(p, tstart, t);
        const int blocks = lin_blocks(p, c);
        const int per = SPLIT ? (blocks + p.split - 1) / p.split : blocks;
        const int kb0 = SPLIT ? static_cast<int>(rank) * per : 0, kb1 = min(blocks, kb0 + per);
        const uint32_t acc = FORM == FORM_WIDE ? sub : p.acc_slots == 2 ? local & 1u : 0u;
        const uint32_t aph = FORM != FORM_WIDE && p.acc_slots == 2 ? (local >> 1) & 1u : local & 1u;
        if (!__all_sync(0xffffffffu, mbar_wait(tempty0 + 8 * acc, aph ^ 1u, &abort_flag))) {
          if (lane == 0) {
            atomicOr(p.status, FTB_DEV_WAIT_TMEMFREE);
            abort_flag = 1;
          }
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + acc * slot_stride + (FORM == FORM_GATED ? sub * static_cast<uint32_t>(p.bn) : 0u);
        uint32_t accumulate = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!ready && !__all_sync(0xffffffffu, mbar_wait(full0 + 8 * s, ph, &abort_flag))) {
            if (lane == 0) {
              atomicOr(p.status, FTB_DEV_WAIT_FULL);
              abort_flag = 1;
            }
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_lo = a_lo0 + off, b_lo = b_lo0 + off;
          // steps of 16 that hold something: the last block of a reduction may have fewer than four
          const int steps = gather_k ? min(4, (c.cnt - kb * kKBlock + 15) >> 4) : 4;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (k < steps) umma<KIND_BF16, PAIR>(d, a_lo + k * a_k, a_hi, b_lo + k * b_k, b_hi, idesc, k > 0 ? 1u : accumulate);
            if constexpr (PAIR) tc_commit_pair_both(empty0 + 8 * s);
            else tc_commit(empty0 + 8 * s);
          }
          __syncwarp();
          {
            // has the next stage landed?
            const uint32_t sn = s + 1 == stages ? 0u : s + 1;
            ready = __all_sync(0xffffffffu, mbar_test_wait(full0 + 8 * sn, sn == 0 ? ph ^ 1u : ph));
          }
          accumulate = 1;
          off += stage_enc;
          if (++s == stages) {
            s = 0;
            ph ^= 1u;
            off = 0;
          }
        }
        if (ok && elect_one()) {
          if constexpr (PAIR) tc_commit_pair_both(tfull0 + 8 * acc);
          else tc_commit(tfull0 + 8 * acc);
        }
        __syncwarp();
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    const int grp = (warp - 4) >> 2, quarter = warp & 3;
    constexpr int GROUPS = EPI / 4;
    const uint32_t tempty_sig = PAIR ? map_to_cta(tempty0, 0) : tempty0;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const long long lane_ldo = p.vec ? (lane >> 2) * p.q.ldo + (lane & 3) * 8 : lane;
    const long long lane_ldp = p.vec ? (lane >> 2) * p.q.ldp + (lane & 3) * 8 : lane;
    int local = 0;
    for (int t = unit; t < total; t += units, ++local) {
      const LinTile c = lin_tile(p, tstart, t);
      const bool work = lin_blocks(p, c) > 0;  // an expert without rows has a gradient of zeros
      // FORM_WIDE: group `grp` of the warps drains sub-tile `grp`
      const uint32_t acc = FORM == FORM_WIDE ? static_cast<uint32_t>(grp) : p.acc_slots == 2 ? local & 1u : 0u;
      const uint32_t aph = FORM != FORM_WIDE && p.acc_slots == 2 ? (local >> 1) & 1u : local & 1u;
      const long long i = static_cast<long long>(c.ti) * p.feat + (FORM == FORM_WIDE ? grp * p.sub_off : 0) +
                          (PAIR ? rank * 128 : 0) + quarter * 32 + lane;
      const bool live = i < p.q.I;
      float b0 = 0.0f, b1 = 0.0f;
      if (!SPLIT && RICH && live && p.q.bias) {
        const uint16_t* bias = p.q.bias + c.g * p.q.bias_gs + i;
        b0 = from16(bias[0], p.q.f16 != 0);
        if (FORM == FORM_GATED) b1 = from16(bias[p.q.I], p.q.f16 != 0);
      }
      const long long j0 = static_cast<long long>(c.tj) * p.bn;
      const int left = static_cast<int>(min((mode == LIN_ROWS ? static_cast<long long>(c.cnt) : p.q.J) - j0,
                                            static_cast<long long>(p.bn)));
      const long long row0 = (mode == LIN_ROWS ? c.lo : 0) + j0;  // (left <= 0: no column is stored)
      const long long out_base = mode == LIN_REDUCE ? c.g * p.q.out_gs : 0;
      constexpr bool GATED = FORM == FORM_GATED;
      const int first = FORM == FORM_WIDE ? 0 : grp * kCols, step = FORM == FORM_WIDE ? kCols : GROUPS * kCols;
      const bool vec = p.vec != 0, add = !SPLIT && RICH && p.q.residual != nullptr;
      WarpCols w;
      w.turn = reinterpret_cast<float*>(smem_raw + (smem_base - smem_u32(smem_raw)) + stages * stage_bytes) + (warp - 4) * kTurnFloats;
      w.lane = lane;
      w.live = live;
      w.live8 = i - lane + (lane & 3) * 8 < p.q.I;
      // this lane's element of the warp's first column in out and residual, and in preact
      long long at = out_base + (row0 + first) * p.q.ldo + (i - lane) + lane_ldo;
      long long zat = (row0 + first) * p.q.ldp + (i - lane) + lane_ldp;
      const long long at_step = step * p.q.ldo, zat_step = step * p.q.ldp;
      uint32_t res[kCols];
      w.valid = left - first;
      if (add) lin_residual(vec, w, res, p.q.residual + at, p.q.ldo);
      const bool got = __all_sync(0xffffffffu, mbar_wait(tfull0 + 8 * acc, aph, &abort_flag));
      if (!got) {
        if (lane == 0) {
          atomicOr(p.status, FTB_DEV_WAIT_TMEMFULL);
          abort_flag = 1;
        }
        if constexpr (SPLIT) {  // the barriers that the other warps and CTAs wait at
          cluster_wait();
          named_barrier_arrive(1, 160);
        }
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem_base + lanes + acc * slot_stride;
      if constexpr (SPLIT) {
        // fp32 partial sums to the CTAs that finish their columns: [source rank][sub][four columns][feature][column]
        const int per = (lin_blocks(p, c) + p.split - 1) / p.split;
        const bool mine = static_cast<int>(rank) * per < lin_blocks(p, c);
        const int share = split_share(left, p.split);
        const uint32_t inbox = smem_base + stages * stage_bytes;
        cluster_wait();  // every CTA of the cluster has started
        for (int sub = 0; sub < SUBS; ++sub)
          for (int c0 = 0; c0 < p.bn && c0 < left; c0 += 16) {
            uint32_t v[16];
            tmem_ld_32x16(d + sub * p.bn + c0, v);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              if (c0 + e < left) {
                const int owner = (c0 + e) / share, quad = ((c0 + e) - owner * share) >> 2;
                const uint32_t to = inbox + ((((rank * SUBS + sub) * (share >> 2) + quad) * 128 + quarter * 32 + lane) << 4);
                st_cluster_f32x4(map_to_cta(to, owner), mine ? __uint_as_float(v[e]) : 0.0f, mine ? __uint_as_float(v[e + 1]) : 0.0f,
                                 mine ? __uint_as_float(v[e + 2]) : 0.0f, mine ? __uint_as_float(v[e + 3]) : 0.0f);
              }
          }
        tc_fence_before();
        named_barrier_arrive(1, 160);  // tensor memory has been read
        break;  // one tile per cluster
      } else {
        uint32_t rv[kCols], ru[kCols];
        auto load = [&](int at) {
          tmem_ld_32x16(d + at, rv);
          if constexpr (GATED) tmem_ld_32x16(d + p.bn + at, ru);
        };
        const int stop = min(p.bn, left);
        if (first < stop) load(first);
        for (int c0 = first; c0 < stop; c0 += step) {
          uint32_t now[kCols];
          float v[kCols], u[kCols];
#pragma unroll
          for (int e = 0; e < kCols; ++e) now[e] = res[e];
          if (add && c0 + step < left) {
            w.valid = left - c0 - step;
            lin_residual(vec, w, res, p.q.residual + at + at_step, p.q.ldo);
          }
          w.valid = left - c0;
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < kCols; ++e) {
            v[e] = __uint_as_float(rv[e]);
            if constexpr (GATED) u[e] = __uint_as_float(ru[e]);
          }
          if (!work) {
#pragma unroll
            for (int e = 0; e < kCols; ++e) v[e] = 0.0f;
          }
          if (c0 + step < stop) load(c0 + step);
          lin_finish<GATED, RICH>(p.q, vec, w, v, u, now, b0, b1, p.q.out + at, p.q.preact + zat);
          at += at_step;
          zat += zat_step;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR) mbar_arrive_cluster(tempty_sig + 8 * acc);
          else mbar_arrive(tempty_sig + 8 * acc);
        }
      }
    }
    __syncwarp();
  }

  if constexpr (SPLIT) {
    // Tensor memory goes back before this CTA waits for its peers: a CTA of another kernel that waits for columns of
    // this SM then never holds up a peer that this cluster waits for.
    if (warp == 1) {
      named_barrier_sync(1, 160);
      tc_fence_after();
      tmem_dealloc(tmem_base, p.tmem_cols);
    }
    if (warp < 4) cluster_wait();  // (the epilogue has waited for the start already)
    __syncwarp();
    cluster_arrive();
    // A CTA finishes a run of the tile's columns, a thread four of one feature at a time; what it adds is asked for
    // before the wait.
    const LinTile c = lin_tile(p, tstart, unit);
    const bool f16 = p.q.f16 != 0;
    const int f = threadIdx.x & 127;
    const long long i = static_cast<long long>(c.ti) * p.feat + f;
    const int left = static_cast<int>(min(p.q.J - static_cast<long long>(c.tj) * p.bn, static_cast<long long>(p.bn)));
    const int share = split_share(left, p.split), first = static_cast<int>(rank) * share, end = min(left, first + share);
    const long long row0 = static_cast<long long>(c.tj) * p.bn;
    int col = first + 4 * (threadIdx.x >> 7);
    float b0 = 0.0f, b1 = 0.0f;
    uint16_t res[4] = {};
    const bool live = i < p.q.I;
    auto residual = [&](int from) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (from + e < end) res[e] = p.q.residual[(row0 + from + e) * p.q.ldo + i];
    };
    if (live && col < end) {
      if (p.q.bias) {
        b0 = from16(p.q.bias[i], f16);
        if (FORM == FORM_GATED) b1 = from16(p.q.bias[p.q.I + i], f16);
      }
      if (p.q.residual) residual(col);
    }
    cluster_wait();  // the partial sums of every CTA are here
    const float4* inbox = reinterpret_cast<const float4*>(smem_raw + (smem_base - smem_u32(smem_raw)) + stages * stage_bytes);
    for (; col < end; col += 8) {
      float sum[2][4] = {};
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub)
        for (int r = 0; r < p.split; ++r) {
          const float4 got = inbox[((r * SUBS + sub) * (share >> 2) + ((col - first) >> 2)) * 128 + f];
          sum[sub][0] += got.x;
          sum[sub][1] += got.y;
          sum[sub][2] += got.z;
          sum[sub][3] += got.w;
        }
      if (!live) continue;
      uint16_t now[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) now[e] = res[e];
      if (p.q.residual && col + 8 < end) residual(col + 8);
      lin_finish4<FORM == FORM_GATED>(p.q, sum[0], sum[1], b0, b1, now, i, row0 + col, end - col);
    }
  }

  // ------------------------------------------------------------ teardown
  if (*reinterpret_cast<volatile int*>(&abort_flag)) {
    // copies still in flight land before shared memory is released
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  if constexpr (SPLIT) return;  // nothing reads or writes this CTA's shared memory any more
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();  // shared memory and TMEM stay until both CTAs are done
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) tmem_dealloc_pair(tmem_base, p.tmem_cols);
    else tmem_dealloc(tmem_base, p.tmem_cols);
  }
}

// ------------------------------------------------------------------ host
constexpr size_t kStaticSmem = 6 * 1024;  // barriers and the tile table
constexpr size_t kOneCta = 227 * 1024 - kStaticSmem;
constexpr size_t kTwoCtas = 113 * 1024 - kStaticSmem;

struct LinPick {
  bool pair;
  int form, bn, split;
  bool deep;  // single CTAs with an SM's shared memory each: no more of them than SMs, and clusters of at most four
              // (eight such CTAs find room in a GPC twice at best: 22 us for 8 x 2048 x 8192, 10.6 with two CTAs an SM)
};

static size_t stage_size(const LinPick& c) {
  return (c.form == FORM_PLAIN ? 1 : 2) * static_cast<size_t>(kSubBytes) + static_cast<size_t>(c.bn / (c.pair ? 2 : 1)) * 128;
}

// Shared memory behind the stages: the epilogue's staging, or the inbox of a split reduction.
static size_t turn_bytes(const LinPick& c) {
  if (c.split > 1) return static_cast<size_t>(c.split) * split_share(c.bn, c.split) * (c.form == FORM_PLAIN ? 1 : 2) * 128 * sizeof(float);
  return static_cast<size_t>(c.pair ? 8 : 4) * kTurnFloats * sizeof(float);
}

static int max_stages(const LinPick& c) {
  size_t n = 0;
  if (!c.pair && !c.deep && kTwoCtas > 1024 + turn_bytes(c)) n = (kTwoCtas - 1024 - turn_bytes(c)) / stage_size(c);
  if (n < 2) n = (kOneCta - 1024 - turn_bytes(c)) / stage_size(c);  // (also where two stages and a wide inbox need it)
  return static_cast<int>(n < kLinStages ? n : kLinStages);
}

// Tiles of a product, at most: a group ends in at most one partial tile.
static int64_t most_tiles(const LinArgs& q, const LinPick& c) {
  const int64_t ti = ceil_div64(q.I, 128 * (c.pair ? 2 : 1) * (c.form == FORM_WIDE ? 2 : 1));
  if (q.mode == LIN_ROWS) return (q.rows / c.bn + (q.groups < q.rows ? q.groups : q.rows)) * ti;
  return ceil_div64(q.J, c.bn) * ti * (q.mode == LIN_REDUCE ? q.groups : 1);
}

// Time of a product under one variant, in SM cycles.  What the terms stand for, with what was measured:
//   a stage costs its rows (128 bytes each) through the SM's port, 2.65 cycles a row, its MMAs, bn / 2 cycles of
//   arithmetic per step of 16 and A sub-tile (1.3 times that with two sub-tiles, which run into the power cap), its share
//   of a copy's latency (2400 cycles over the stages in flight, half a stage less), or the hand-offs of one stage (500
//   cycles in a pair, 420 alone), whichever is most; rows fetched by number cost 12 cycles each;
//   no product is faster than its operands and results at the 3450 bytes a cycle of the memory;
//   the epilogue costs a scheduler's warps in turn about 22 cycles per column, 16 more for an activation, 6 for a residual
//   and for preact, half as many again in 2-byte accesses; it runs under the next tile's main loop where a second
//   accumulator exists;
//   a split reduction costs two cluster barriers and the exchange of its columns.
// What it has to tell apart, measured: 1 x 4096 x 4096 split 8 / 4 / 2: 11.7 / 9.7 / 13.6 us; 256 x 4096 x 4096 pairs of
// 64 / 128 / 256 tokens 23.3 / 23.9 / 25.3; 1237 x 2048 x 1000 with a rich epilogue, pairs of 160 / 256 tokens 15.6 / 20.1,
// single CTAs of 128 tokens 24.4.
static double variant_cycles(const LinArgs& q, LinPick c, int sms) {
  c.deep = !c.pair && c.split <= 4 && most_tiles(q, c) * c.split <= sms;
  const double blocks = q.mode == LIN_REDUCE ? static_cast<double>(q.rows) / q.groups / kKBlock + 0.5
                                             : static_cast<double>(ceil_div64(q.K, kKBlock));
  const int subs = c.form == FORM_PLAIN ? 1 : 2, mult = (c.pair ? 2 : 1) * (c.form == FORM_WIDE ? 2 : 1);
  const double tiles_i = static_cast<double>(ceil_div64(q.I, 128 * mult));
  const double busy = static_cast<double>(q.groups < q.rows ? q.groups : q.rows);
  double tiles;
  if (q.mode == LIN_ROWS) {
    // the rows of a group fill its tiles but for half of the last one
    tiles = static_cast<double>(q.rows) / c.bn + 0.5 * busy;
    if (tiles < busy) tiles = busy;
  } else {
    tiles = static_cast<double>(ceil_div64(q.J, c.bn)) * (q.mode == LIN_REDUCE ? q.groups : 1);
  }
  tiles *= tiles_i * c.split;
  const int per_sm = !c.pair && tiles > sms ? 2 : 1;
  const double units = c.pair ? sms / 2 : sms * per_sm;
  double waves = tiles / units;
  if (q.mode != LIN_ROWS || waves < 1) waves = static_cast<double>(static_cast<int64_t>(waves + 0.999999));
  else waves += 0.5;
  const int bj = c.pair ? c.bn / 2 : c.bn;
  double load = 2.65 * (128 * subs + bj);
  if (q.mode == LIN_ROWS && q.gather_div) load += (12 - 2.65) * bj;
  const double latency = 2400.0 / (max_stages(c) - 0.5), handoff = c.pair ? 500 : 420;
  const double math = (subs == 2 ? 1.3 : 1.0) * 4.0 * subs * (c.bn / 2 > 64 ? c.bn / 2 : 64);
  double stage = (load > math ? load : math) * per_sm;
  if (stage < latency) stage = latency;
  if (stage < handoff) stage = handoff;
  const double main_loop = static_cast<double>(static_cast<int64_t>(blocks / c.split + 0.999999)) * stage;
  double per_col = 22 + (q.act ? 16 : 0) + (q.residual ? 6 : 0) + (q.preact ? 6 * subs : 0) + (q.gated ? 8 : 0);
  if (q.I % 8) per_col *= 1.5;
  // a pair's eight warps share the columns, or each sub-tile's four take all of them
  const double epi = c.pair ? per_col * (c.form == FORM_WIDE ? 2 * c.bn : c.bn) : per_col * c.bn * per_sm;
  const bool covered = c.form == FORM_PLAIN || (c.form == FORM_GATED && (c.pair ? c.bn <= 128 : c.bn <= 64));
  const double tile = covered ? (main_loop > epi ? main_loop : epi) : main_loop + epi;
  double body = (waves - 1) * tile + main_loop;
  const double a_bytes = 2.0 * q.I * (q.gated ? 2 : 1) * (q.mode == LIN_REDUCE ? q.rows : q.K) * (q.mode == LIN_ROWS ? busy : 1);
  const double memory = (a_bytes + 2.0 * q.J * q.I) / 3450;
  if (body < memory) body = memory;
  double total = 3000 + body + epi;
  if (c.split > 1) total += 5000 + 220.0 * subs * (q.J < c.bn ? q.J : c.bn) / c.split;
  return total;
}

// Variant for a product: the cheapest by the estimate above.
static LinPick pick_variant(const LinArgs& q, int sms) {
  LinPick best;
  memset(&best, 0, sizeof(best));
  double least = 1e300;
  auto consider = [&](bool pair, int form, int bn, int split) {
    LinPick c;
    memset(&c, 0, sizeof(c));
    c.pair = pair;
    c.form = form;
    c.bn = bn;
    c.split = split;
    const double t = variant_cycles(q, c, sms);
    if (t < least) {
      least = t;
      best = c;
    }
  };
  const int64_t most = q.mode == LIN_ROWS ? q.rows : q.J;  // no group has more tokens
  const int step = q.b_mn ? 64 : 16;                       // an MN-major B is staged in blocks of 64
  const int64_t blocks = ceil_div64(q.K, kKBlock);
  for (int bn = step; bn <= 128; bn += bn < 64 ? step : 32) {
    if (q.b_mn && bn % 64) continue;
    const int form = q.gated ? FORM_GATED : FORM_PLAIN;
    consider(false, form, bn, 1);
    const int64_t tiles = ceil_div64(q.I, 128) * ceil_div64(q.J, bn);
    if (q.mode == LIN_DENSE && bn <= 64)
      for (int split = 2; split <= 8 && tiles * split <= 2 * sms && blocks >= 2 * split; split *= 2) consider(false, form, bn, split);
    if (bn >= most) break;
  }
  if (most > 64 && sms >= 2)
    for (int bn = 2 * step > 64 ? 2 * step : 64; bn <= 256; bn += q.b_mn ? 128 : 32) {
      if (q.gated) {
        consider(true, FORM_GATED, bn, 1);
      } else {
        consider(true, FORM_PLAIN, bn, 1);
        consider(true, FORM_WIDE, bn, 1);
      }
      if (bn >= most) break;
    }
  return best;
}

template <bool PAIR, int FORM, int EPI, bool SPLIT, bool RICH>
static int launch_variant(const LinMaps& maps, const LinUmma& p, int ctas, size_t smem, cudaStream_t stream) {
  auto kern = linear_umma_kernel<PAIR, FORM, EPI, SPLIT, RICH>;
  static std::mutex mu;
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 0 && dev < 64 && !done[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kOneCta));
      if (e != cudaSuccess) return launch_status(e);
      done[dev] = true;
    }
  }
  return launch_overlapped(kern, dim3(static_cast<unsigned>(ctas)), dim3(128 + 32 * EPI), smem, PAIR ? 2 : SPLIT ? p.split : 1,
                           stream, maps, p);
}

int launch_linear_umma(const LinArgs& q, const ftb_config* cfg, int* status, cudaStream_t stream) {
  // TMA addresses 16-byte rows and bases only
  if ((q.lda * 2) % 16 || (q.ldb * 2) % 16 || (reinterpret_cast<uintptr_t>(q.a) & 15) || (reinterpret_cast<uintptr_t>(q.b) & 15))
    return FTB_E_UNSUPPORTED;
  const int sms = sm_count();
  LinPick c = pick_variant(q, sms);
  if (cfg) {
    if (cfg->tile_n || cfg->cluster || cfg->split_k) {
      const bool pair = cfg->cluster ? cfg->cluster == 2 : cfg->tile_n ? cfg->tile_n == 256 : cfg->split_k > 1 ? false : c.pair;
      if (pair != c.pair) c.form = q.gated ? FORM_GATED : FORM_PLAIN;
      c.pair = pair;
      if (cfg->tile_n) c.bn = cfg->tile_n;
      if (pair && c.bn < 64) c.bn = 128;
      if (!pair && c.bn > 128) c.bn = 128;
      if (cfg->split_k) {
        c.split = cfg->split_k;
        if (c.split > 1 && c.bn > 64) c.bn = 64;
      } else if (pair || c.bn > 64) {
        c.split = 1;
      }
    }
  }
  const int64_t most = most_tiles(q, c);
  if (most > 0x7fffffffll / 8) return FTB_E_TOO_LARGE;
  c.deep = !c.pair && c.split <= 4 && most * c.split <= sms;
  const bool two = !c.pair && !c.deep;
  int stages = max_stages(c);
  if (cfg && cfg->stages) {
    if (cfg->stages > stages) return FTB_E_BAD_CONFIG;
    stages = cfg->stages;
  }
  if (stages < 2) return FTB_E_BAD_CONFIG;

  LinUmma p;
  memset(&p, 0, sizeof(p));
  p.q = q;
  const int subs = c.form == FORM_PLAIN ? 1 : 2, m = c.pair ? 256 : 128;
  p.bn = c.bn;
  p.bj = c.pair ? c.bn / 2 : c.bn;
  p.stages = stages;
  p.split = c.split;
  p.feat = c.form == FORM_WIDE ? 2 * m : m;
  p.sub_off = c.form == FORM_WIDE ? m : static_cast<int>(q.I);
  p.tiles_i = static_cast<int>(ceil_div64(q.I, p.feat));
  p.tiles_j = static_cast<int>(q.mode == LIN_ROWS ? 1 : ceil_div64(q.J, c.bn));
  p.most_rows = static_cast<int>(most / p.tiles_i);
  p.band = 8;
  p.by_i = fast_div(p.tiles_i);
  p.by_group = fast_div(static_cast<int64_t>(p.tiles_i) * p.tiles_j);
  p.by_span = fast_div(static_cast<int64_t>(p.tiles_i) * p.band);
  p.by_band = fast_div(p.band);
  p.by_last = fast_div(p.tiles_j % p.band ? p.tiles_j % p.band : p.band);
  const int acc_cols = subs * c.bn;
  p.acc_slots = c.form == FORM_WIDE ? 2 : c.split > 1 || 2 * acc_cols > (c.pair ? 512 : 256) ? 1 : 2;
  uint32_t cols = 32;
  while (cols < static_cast<uint32_t>(c.form == FORM_WIDE ? acc_cols : p.acc_slots * acc_cols)) cols *= 2;
  p.tmem_cols = cols;
  // instruction descriptor: fp32 accumulator, both operands bf16 (1) or both fp16 (0)
  const uint32_t fmt = q.f16 ? 0u : 1u;
  p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(q.a_mn) << 15) |
            (static_cast<uint32_t>(q.b_mn) << 16) | (static_cast<uint32_t>(c.bn >> 3) << 17) |
            (static_cast<uint32_t>(m >> 4) << 24);
  // k-contiguous rows of 128 bytes, or 64-element blocks of i (j) with one row per k
  p.a_lbo = q.a_mn ? 8192 : 16;
  p.b_lbo = q.b_mn ? 8192 : 16;
  p.a_kadv = q.a_mn ? 2048 : 32;
  p.b_kadv = q.b_mn ? 2048 : 32;
  const uintptr_t rows16 = reinterpret_cast<uintptr_t>(q.out) | reinterpret_cast<uintptr_t>(q.residual) | reinterpret_cast<uintptr_t>(q.preact);
  p.vec = (rows16 & 15) == 0 && q.I % 8 == 0 && q.ldo % 8 == 0 && q.ldp % 8 == 0 && q.out_gs % 8 == 0;
  p.status = status ? status : fallback_status();
  if (!p.status) return FTB_E_CUDA;

  const CUtensorMapDataType dt = q.f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint32_t ones[3] = {1, 1, 1};
  LinMaps maps;
  memset(&maps, 0, sizeof(maps));
  const bool reduce = q.mode == LIN_REDUCE, gathers = q.gather_div != 0;
  int rc = FTB_OK;
  {
    // A: [group][row][k], or [group][k][i]; a reduction has one matrix of places
    const uint64_t a_rows = static_cast<uint64_t>(q.gated ? 2 * q.I : q.I), kk = static_cast<uint64_t>(reduce ? q.rows : q.K);
    const uint64_t d[3] = {q.a_mn ? a_rows : kk, q.a_mn ? kk : a_rows, static_cast<uint64_t>(q.mode == LIN_ROWS ? q.groups : 1)};
    const uint32_t box[3] = {64, q.a_mn ? 64u : 128u, 1};
    const uint64_t st[2] = {static_cast<uint64_t>(q.lda) * 2, d[1] * static_cast<uint64_t>(q.lda) * 2};
    rc = make_tmap(&maps.a, dt, 3, q.a, d, st, box, ones);
    if (!rc && reduce) {
      const uint32_t row_box[2] = {64, 1}, run_box[3] = {64, 16, 1};
      rc = make_tmap(&maps.a_rows, dt, 2, q.a, d, st, row_box, ones);
      if (!rc) rc = make_tmap(&maps.a16, dt, 3, q.a, d, st, run_box, ones);
    }
    if (rc) return rc;
  }
  {
    const uint64_t rows = static_cast<uint64_t>(q.mode == LIN_ROWS ? (gathers ? q.src_rows : q.rows) : q.J);
    const uint64_t kk = static_cast<uint64_t>(reduce ? q.rows : q.K);
    const uint64_t d[3] = {q.b_mn ? rows : kk, q.b_mn ? kk : rows, 1};
    const uint32_t box[3] = {64, q.b_mn ? 64u : static_cast<uint32_t>(p.bj), 1};
    const uint64_t st[2] = {static_cast<uint64_t>(q.ldb) * 2, d[1] * static_cast<uint64_t>(q.ldb) * 2};
    if (!(q.mode == LIN_ROWS && gathers)) rc = make_tmap(&maps.b, dt, 3, q.b, d, st, box, ones);
    if (!rc && (reduce || (q.mode == LIN_ROWS && gathers))) {
      const uint32_t row_box[2] = {64, 1}, run_box[3] = {64, 16, 1};
      rc = make_tmap(&maps.b_rows, dt, 2, q.b, d, st, row_box, ones);
      if (!rc && reduce) rc = make_tmap(&maps.b16, dt, 3, q.b, d, st, run_box, ones);
      p.oob_b = static_cast<int>(d[1]);
    }
    if (rc) return rc;
  }

  size_t smem = static_cast<size_t>(stages) * stage_size(c) + 1024 + turn_bytes(c);
  if (c.pair) smem = pair_shared_bytes(smem);
  const bool rich = q.gated || q.act || q.bias || q.residual || q.preact;
  if (c.split > 1) {
    const int ctas = static_cast<int>(most) * c.split;
    return c.form == FORM_GATED ? launch_variant<false, FORM_GATED, 4, true, true>(maps, p, ctas, smem, stream)
                                : launch_variant<false, FORM_PLAIN, 4, true, true>(maps, p, ctas, smem, stream);
  }
  if (c.pair) {
    const int64_t units = sms / 2 < most ? sms / 2 : most;
    const int ctas = static_cast<int>(units) * 2;
    if (c.form == FORM_GATED) return launch_variant<true, FORM_GATED, 8, false, true>(maps, p, ctas, smem, stream);
    if (c.form == FORM_WIDE)
      return rich ? launch_variant<true, FORM_WIDE, 8, false, true>(maps, p, ctas, smem, stream)
                  : launch_variant<true, FORM_WIDE, 8, false, false>(maps, p, ctas, smem, stream);
    return rich ? launch_variant<true, FORM_PLAIN, 8, false, true>(maps, p, ctas, smem, stream)
                : launch_variant<true, FORM_PLAIN, 8, false, false>(maps, p, ctas, smem, stream);
  }
  const int64_t slots = two ? 2 * sms : sms;
  const int ctas = static_cast<int>(slots < most ? slots : most);
  if (c.form == FORM_GATED) return launch_variant<false, FORM_GATED, 4, false, true>(maps, p, ctas, smem, stream);
  return rich ? launch_variant<false, FORM_PLAIN, 4, false, true>(maps, p, ctas, smem, stream)
              : launch_variant<false, FORM_PLAIN, 4, false, false>(maps, p, ctas, smem, stream);
}

}  // namespace ftb
