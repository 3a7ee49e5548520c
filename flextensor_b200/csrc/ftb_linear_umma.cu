// The products with an epilogue on tcgen05: out[j, i] = epilogue(sum over k of A[i, k] B[j, k]).
//
// Features (i) lie on the 128 lanes of tensor memory and tokens (j) on its columns, in every direction: a tile of few
// tokens is then a narrow accumulator (16 columns for one token) instead of 128 mostly empty rows, a thread of the
// epilogue owns one feature, so its bias is one register, and 32 lanes store 32 neighbouring features of a token.
//
//   warp 0      producer: TMA tiles of A and B into 128-byte swizzled stages of 64 k; rows named by a list (tokens of
//               an expert, or the reduction of its weight gradient) come by gather4, four rows per lane and copy, and a
//               row past the end of its expert is asked for outside the tensor, which fills it with zeros
//   warp 1, 2   issuers of tcgen05.mma, one per A sub-tile (one thread issues an MMA every 137 cycles at best)
//   warps 4..   epilogue: tcgen05.ld -> bias, activation, gate, residual -> 2-byte stores, 64 bytes per warp
//
// Forms: FORM_PLAIN one A sub-tile; FORM_GATED two, the gate rows and the others of the same features, whose
// accumulators share lanes and columns, so the gate is applied in registers; FORM_WIDE two neighbouring feature tiles
// over the same tokens (a byte of B feeds twice the math).  PAIR runs two CTAs as one cta_group::2 unit.
// SPLIT gives the reduction of one tile to the CTAs of a cluster, which add their fp32 partial sums through
// distributed shared memory in rank order.
//
// Waits are bounded as in ftb_umma_kernel.cuh: a role that gives up sets a status bit and the CTA leaves through its
// normal teardown.
#include "ftb_linear.h"
#include "ftb_ptx.cuh"
#include "ftb_tmap.h"

#include <mutex>

namespace ftb {

enum { FORM_PLAIN = 0, FORM_GATED = 1, FORM_WIDE = 2 };
constexpr int kLinStages = 8;
constexpr uint32_t kSubBytes = 128 * 128;  // 128 rows x 64 elements
constexpr int kKBlock = 64;

struct LinUmma {
  LinArgs q;
  int bn, bj;            // tokens per tile, and of those staged per CTA
  int stages, split;
  int tiles_i, tiles_j;  // tiles_j: LIN_DENSE and LIN_REDUCE
  int feat, sub_off;     // features per tile; feature rows between the A sub-tiles
  int band;              // token tiles walked together before the next feature tile
  int acc_slots;         // accumulators in turn (FORM_WIDE: one per sub-tile)
  uint32_t tmem_cols;
  uint32_t idesc;
  uint32_t a_lbo, b_lbo, a_kadv, b_kadv;
  int oob_a, oob_b;      // a row past the gathered tensors
  int* status;
};

struct LinTile {
  int g, ti, tj, lo, cnt;  // group, feature tile, token tile; the group's first place and number of places
};

__device__ __forceinline__ LinTile lin_tile(const LinUmma& p, const int* tstart, int t) {
  LinTile c;
  c.g = 0;
  c.lo = 0;
  c.cnt = 0;
  if (p.q.mode == LIN_ROWS) {
    // the group whose run of tiles holds t
    int a = 0, b = p.q.groups;
    while (b - a > 1) {
      const int mid = (a + b) >> 1;
      if (static_cast<long long>(tstart[mid]) * p.tiles_i <= t) a = mid;
      else b = mid;
    }
    c.g = a;
    const int nj = tstart[a + 1] - tstart[a], r = t - tstart[a] * p.tiles_i;
    c.ti = r / nj;
    c.tj = r - c.ti * nj;
    int hi;
    group_range(p.q.offsets, a, p.q.rows, &c.lo, &hi);
    c.cnt = hi - c.lo;
    return c;
  }
  const int per = p.tiles_i * p.tiles_j;
  int r = t;
  if (p.q.mode == LIN_REDUCE) {
    c.g = t / per;
    r = t - c.g * per;
    int hi;
    group_range(p.q.offsets, c.g, p.q.rows, &c.lo, &hi);
    c.cnt = hi - c.lo;
  }
  // bands of `band` token tiles: inside one, token tiles run fastest
  const int span = p.band * p.tiles_i, b = r / span, first = b * p.band;
  const int width = min(p.band, p.tiles_j - first), q = r - b * span;
  c.ti = q / width;
  c.tj = first + q - c.ti * width;
  return c;
}

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

// bias, activation, gate, residual and the stores of `NC` neighbouring tokens of one feature; `at` is its element of the
// first token in out and residual, `zat` in preact.
template <int NC, bool GATED>
__device__ __forceinline__ void lin_finish(const LinArgs& q, float (&v)[NC], float (&u)[NC], float b0, float b1,
                                           long long at, long long zat, int valid) {
  const bool f16 = q.f16 != 0;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    v[c] += b0;
    if constexpr (GATED) u[c] += b1;
  }
  if (q.preact) {
    uint16_t* z = q.preact + zat;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (c < valid) {
        *z = to16(v[c], f16);
        if constexpr (GATED) z[q.I] = to16(u[c], f16);
      }
      z += q.ldp;
    }
  }
  act_values<NC>(v, q.act);
  if constexpr (GATED) {
#pragma unroll
    for (int c = 0; c < NC; ++c) v[c] *= u[c];
  }
  if (q.residual) {
    const uint16_t* r = q.residual + at;
    uint16_t res[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      res[c] = c < valid ? *r : 0;
      r += q.ldo;
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) v[c] += from16(res[c], f16);
  }
  uint16_t* out = q.out + at;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (c < valid) *out = to16(v[c], f16);
    out += q.ldo;
  }
}

template <bool PAIR, int FORM, int EPI, bool SPLIT>
__global__ void __launch_bounds__(128 + 32 * EPI, EPI == 4 ? 2 : 1)
linear_umma_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ LinUmma p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kLinStages];
  __shared__ __align__(8) uint64_t bar_empty[kLinStages];
  __shared__ __align__(8) uint64_t bar_tfull[2];
  __shared__ __align__(8) uint64_t bar_tempty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ int tstart[FTB_MAX_EXPERTS + 1];
  constexpr int SUBS = FORM == FORM_PLAIN ? 1 : 2;
  static_assert(!SPLIT || (!PAIR && FORM != FORM_WIDE && EPI == 4), "the reduction is split in single-CTA tiles only");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t b_bytes = static_cast<uint32_t>(p.bj) * 128u;
  const uint32_t stage_bytes = SUBS * kSubBytes + b_bytes;
  const uint32_t rank = (PAIR || SPLIT) ? cluster_ctarank() : 0u;
  const int unit = PAIR ? blockIdx.x >> 1 : SPLIT ? blockIdx.x / p.split : blockIdx.x;
  const int units = PAIR ? gridDim.x >> 1 : SPLIT ? gridDim.x / p.split : gridDim.x;
  const uint32_t stages = p.stages;
  const int mode = p.q.mode;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (uint32_t s = 0; s < stages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);
      mbar_init(smem_u32(&bar_empty[s]), SUBS);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&bar_tfull[a]), FORM == FORM_GATED ? 2 : 1);
      mbar_init(smem_u32(&bar_tempty[a]), (FORM == FORM_WIDE ? EPI / 2 : EPI) * (PAIR ? 2 : 1));
    }
    fence_mbar_init();
    fence_proxy_async_smem();
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_b);
  }
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
      if (g0 + lane < p.q.groups) tstart[g0 + lane + 1] = base + x;
      base += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) tstart[0] = 0;
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();  // the peer's barriers exist before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;

  const int total = mode == LIN_ROWS ? tstart[p.q.groups] * p.tiles_i : p.q.groups * p.tiles_i * p.tiles_j;
  const uint32_t full0 = smem_u32(&bar_full[0]), empty0 = smem_u32(&bar_empty[0]);
  const uint32_t tfull0 = smem_u32(&bar_tfull[0]), tempty0 = smem_u32(&bar_tempty[0]);
  const uint32_t slot_stride = FORM == FORM_WIDE ? static_cast<uint32_t>(p.bn) : static_cast<uint32_t>(p.bn) * SUBS;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    const bool gather_j = mode == LIN_ROWS && p.q.gather_div != 0;
    const bool gather_k = mode == LIN_REDUCE;
    const bool gather = gather_j || gather_k;
    const unsigned takers = gather ? 0xffffffffu : 1u;  // lanes of this loop
    if (lane == 0 || gather) {
      const uint32_t tx = stage_bytes;
      const uint32_t sig0 = PAIR ? map_to_cta(full0, 0) : full0;
      uint32_t s = 0, ph = 0, sa = smem_base;
      bool ok = true;
      for (int t = unit; t < total && ok; t += units) {
        const LinTile c = lin_tile(p, tstart, t);
        const int blocks = lin_blocks(p, c);
        const int per = SPLIT ? (blocks + p.split - 1) / p.split : blocks;
        const int kb0 = SPLIT ? static_cast<int>(rank) * per : 0, kb1 = min(blocks, kb0 + per);
        const int f0 = c.ti * p.feat + static_cast<int>(rank) * (PAIR ? 128 : 0);
        const int j0 = c.tj * p.bn + static_cast<int>(rank) * (PAIR ? p.bj : 0);
        int row[4] = {};
        if (gather_j && lane * 4 < p.bj) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = j0 + lane * 4 + e;
            const long long r = j < c.cnt ? gathered_row(p.q, c.lo + j) : -1;
            row[e] = r >= 0 ? static_cast<int>(r) : p.oob_b;
          }
        }
        for (int kb = kb0; kb < kb1; ++kb) {
          int ra[4], rb[4];
          if (gather_k) {
            // this lane's four places of the block: 16 lanes cover its 64
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int k = kb * kKBlock + (lane & 15) * 4 + e;
              const long long r = k < c.cnt ? gathered_row(p.q, c.lo + k) : -1;
              ra[e] = r >= 0 ? static_cast<int>(r) : p.oob_a;
              rb[e] = k < c.cnt ? c.lo + k : p.oob_b;
            }
          }
          const bool free = mbar_wait(empty0 + 8 * s, ph ^ 1u, &abort_flag);
          if (!__all_sync(takers, free)) {
            if (lane == 0) {
              atomicOr(p.status, FTB_DEV_WAIT_EMPTY);
              abort_flag = 1;
            }
            ok = false;
            break;
          }
          const uint32_t full = sig0 + 8 * s, sb = sa + SUBS * kSubBytes;
          const int kc = kb * kKBlock;
          if (lane == 0 && rank * (PAIR ? 1u : 0u) == 0u) mbar_expect_tx(full0 + 8 * s, PAIR ? 2 * tx : tx);
          if (gather_k) {
            __syncwarp();
            const int box = lane >> 4;
            const uint32_t at = static_cast<uint32_t>(lane & 15) * 512u;
#pragma unroll
            for (int sub = 0; sub < SUBS; ++sub) {
              const uint32_t dst = sa + sub * kSubBytes + box * 8192u + at;
              const int col = f0 + sub * p.sub_off + box * 64;
              if constexpr (PAIR) tma_gather4_pair(dst, &map_a, full, col, ra[0], ra[1], ra[2], ra[3]);
              else tma_gather4(dst, &map_a, full, col, ra[0], ra[1], ra[2], ra[3]);
            }
            if (box * 64 < p.bj) {
              if constexpr (PAIR) tma_gather4_pair(sb + box * 8192u + at, &map_b, full, j0 + box * 64, rb[0], rb[1], rb[2], rb[3]);
              else tma_gather4(sb + box * 8192u + at, &map_b, full, j0 + box * 64, rb[0], rb[1], rb[2], rb[3]);
            }
          } else {
            if (lane == 0) {
#pragma unroll
              for (int sub = 0; sub < SUBS; ++sub) {
                const uint32_t dst = sa + sub * kSubBytes;
                const int f = f0 + sub * p.sub_off;
                if (p.q.a_mn) {
#pragma unroll
                  for (int b = 0; b < 2; ++b) {
                    if constexpr (PAIR) tma_load_3d_pair(dst + b * 8192u, &map_a, full, f + b * 64, kc, c.g);
                    else tma_load_3d(dst + b * 8192u, &map_a, full, f + b * 64, kc, c.g);
                  }
                } else {
                  if constexpr (PAIR) tma_load_3d_pair(dst, &map_a, full, kc, f, c.g);
                  else tma_load_3d(dst, &map_a, full, kc, f, c.g);
                }
              }
              if (p.q.b_mn) {
                for (int b = 0; b * 64 < p.bj; ++b) {
                  if constexpr (PAIR) tma_load_3d_pair(sb + b * 8192u, &map_b, full, j0 + b * 64, kc, 0);
                  else tma_load_3d(sb + b * 8192u, &map_b, full, j0 + b * 64, kc, 0);
                }
              } else if (!gather_j) {
                if constexpr (PAIR) tma_load_3d_pair(sb, &map_b, full, kc, c.lo + j0, 0);
                else tma_load_3d(sb, &map_b, full, kc, c.lo + j0, 0);
              }
            }
            if (gather_j) {
              __syncwarp();
              if (lane * 4 < p.bj) {
                if constexpr (PAIR) tma_gather4_pair(sb + lane * 512u, &map_b, full, kc, row[0], row[1], row[2], row[3]);
                else tma_gather4(sb + lane * 512u, &map_b, full, kc, row[0], row[1], row[2], row[3]);
              }
            }
          }
          sa += stage_bytes;
          if (++s == stages) {
            s = 0;
            ph ^= 1u;
            sa = smem_base;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1 || (SUBS == 2 && warp == 2)) {
    // ------------------------------------------------------------ MMA issuers (leader CTA of a pair)
    const uint32_t sub = warp - 1;
    if (lane == 0 && (!PAIR || rank == 0)) {
      const uint32_t idesc = p.idesc;
      const uint32_t a_hi = smem_desc_hi(p.a_lbo, 1024, 2), b_hi = smem_desc_hi(p.b_lbo, 1024, 2);
      const uint32_t a_lo0 = smem_desc_lo(smem_base + sub * kSubBytes, p.a_lbo);
      const uint32_t b_lo0 = smem_desc_lo(smem_base + SUBS * kSubBytes, p.b_lbo);
      const uint32_t a_k = p.a_kadv >> 4, b_k = p.b_kadv >> 4, stage_enc = stage_bytes >> 4;
      uint32_t s = 0, ph = 0, off = 0, ready = 0;
      int local = 0;
      bool ok = true;
      for (int t = unit; t < total && ok; t += units, ++local) {
        const LinTile c = lin_tile(p, tstart, t);
        const int blocks = lin_blocks(p, c);
        const int per = SPLIT ? (blocks + p.split - 1) / p.split : blocks;
        const int kb0 = SPLIT ? static_cast<int>(rank) * per : 0, kb1 = min(blocks, kb0 + per);
        const uint32_t acc = FORM == FORM_WIDE ? sub : p.acc_slots == 2 ? local & 1u : 0u;
        const uint32_t aph = FORM != FORM_WIDE && p.acc_slots == 2 ? (local >> 1) & 1u : local & 1u;
        if (!mbar_wait(tempty0 + 8 * acc, aph ^ 1u, &abort_flag)) {
          atomicOr(p.status, FTB_DEV_WAIT_TMEMFREE);
          abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + acc * slot_stride + (FORM == FORM_GATED ? sub * static_cast<uint32_t>(p.bn) : 0u);
        uint32_t accumulate = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!ready && !mbar_wait(full0 + 8 * s, ph, &abort_flag)) {
            atomicOr(p.status, FTB_DEV_WAIT_FULL);
            abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          {
            // has the next stage landed?  (the answer is used in the next iteration)
            const uint32_t sn = s + 1 == stages ? 0u : s + 1;
            ready = mbar_test_wait(full0 + 8 * sn, sn == 0 ? ph ^ 1u : ph);
          }
          const uint32_t a_lo = a_lo0 + off, b_lo = b_lo0 + off;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma<KIND_BF16, PAIR>(d, a_lo + k * a_k, a_hi, b_lo + k * b_k, b_hi, idesc, k > 0 ? 1u : accumulate);
          accumulate = 1;
          if constexpr (PAIR) tc_commit_pair_both(empty0 + 8 * s);
          else tc_commit(empty0 + 8 * s);
          off += stage_enc;
          if (++s == stages) {
            s = 0;
            ph ^= 1u;
            off = 0;
          }
        }
        if (ok) {
          if constexpr (PAIR) tc_commit_pair_both(tfull0 + 8 * acc);
          else tc_commit(tfull0 + 8 * acc);
        }
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    const int grp = (warp - 4) >> 2, quarter = warp & 3;
    constexpr int GROUPS = EPI / 4;
    const uint32_t tempty_sig = PAIR ? map_to_cta(tempty0, 0) : tempty0;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
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
      if (!SPLIT && live && p.q.bias) {
        const uint16_t* bias = p.q.bias + c.g * p.q.bias_gs + i;
        b0 = from16(bias[0], p.q.f16 != 0);
        if (FORM == FORM_GATED) b1 = from16(bias[p.q.I], p.q.f16 != 0);
      }
      const long long j0 = static_cast<long long>(c.tj) * p.bn;
      const int left = static_cast<int>(min((mode == LIN_ROWS ? static_cast<long long>(c.cnt) : p.q.J) - j0,
                                            static_cast<long long>(p.bn)));
      const long long row0 = (mode == LIN_ROWS ? c.lo : 0) + j0;
      const long long out_base = mode == LIN_REDUCE ? c.g * p.q.out_gs : 0;
      const bool got = __all_sync(0xffffffffu, mbar_wait(tfull0 + 8 * acc, aph, &abort_flag));
      if (!got) {
        if (lane == 0) {
          atomicOr(p.status, FTB_DEV_WAIT_TMEMFULL);
          abort_flag = 1;
        }
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem_base + lanes + acc * slot_stride;
      if constexpr (SPLIT) {
        // fp32 partial sums into the (now idle) stages, [sub][column][lane]
        float* part = reinterpret_cast<float*>(smem_raw + (smem_base - smem_u32(smem_raw)));
        const int per = (lin_blocks(p, c) + p.split - 1) / p.split;
        const bool mine = static_cast<int>(rank) * per < lin_blocks(p, c);
        for (int sub = 0; sub < SUBS; ++sub)
          for (int c0 = 0; c0 < p.bn; c0 += 16) {
            uint32_t v[16];
            tmem_ld_32x16(d + sub * p.bn + c0, v);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e)
              part[(sub * p.bn + c0 + e) * 128 + quarter * 32 + lane] = mine ? __uint_as_float(v[e]) : 0.0f;
          }
        break;  // one tile per cluster
      } else {
        constexpr bool GATED = FORM == FORM_GATED;
        const int first = FORM == FORM_WIDE ? 0 : grp, step = FORM == FORM_WIDE ? 1 : GROUPS;
        if (p.bn >= 32) {
          for (int c0 = first * 32; c0 < p.bn && c0 < left; c0 += step * 32) {
            uint32_t rv[32], ru[32];
            float v[32], u[32];
            tmem_ld_32x32(d + c0, rv);
            if constexpr (GATED) tmem_ld_32x32(d + p.bn + c0, ru);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              v[e] = work ? __uint_as_float(rv[e]) : 0.0f;
              if constexpr (GATED) u[e] = __uint_as_float(ru[e]);
            }
            if (live)
              lin_finish<32, GATED>(p.q, v, u, b0, b1, out_base + (row0 + c0) * p.q.ldo + i, (row0 + c0) * p.q.ldp + i, left - c0);
          }
        } else if (first == 0) {
          uint32_t rv[16], ru[16];
          float v[16], u[16];
          tmem_ld_32x16(d, rv);
          if constexpr (GATED) tmem_ld_32x16(d + p.bn, ru);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            v[e] = work ? __uint_as_float(rv[e]) : 0.0f;
            if constexpr (GATED) u[e] = __uint_as_float(ru[e]);
          }
          if (live) lin_finish<16, GATED>(p.q, v, u, b0, b1, out_base + row0 * p.q.ldo + i, row0 * p.q.ldp + i, left);
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
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tmem_base, p.tmem_cols);
    }
    __syncwarp();
    cluster_sync_all();  // every CTA's partial sums are in its shared memory
    if (unit < total) {
      const LinTile c = lin_tile(p, tstart, unit);
      const int f = threadIdx.x & 127;
      const long long i = static_cast<long long>(c.ti) * p.feat + f;
      const long long j0 = static_cast<long long>(c.tj) * p.bn;
      const int left = static_cast<int>(min(p.q.J - j0, static_cast<long long>(p.bn)));
      const bool f16 = p.q.f16 != 0;
      if (i < p.q.I) {
        float b0 = 0.0f, b1 = 0.0f;
        if (p.q.bias) {
          b0 = from16(p.q.bias[i], f16);
          if (FORM == FORM_GATED) b1 = from16(p.q.bias[p.q.I + i], f16);
        }
        // columns are dealt to the CTAs and to the two halves of their threads
        for (int col = static_cast<int>(rank) * 2 + (threadIdx.x >> 7); col < left; col += 2 * p.split) {
          float sum[2][1] = {{0.0f}, {0.0f}};
#pragma unroll
          for (int sub = 0; sub < SUBS; ++sub) {
            const uint32_t at = smem_base + ((sub * p.bn + col) * 128 + f) * 4;
            for (int r = 0; r < p.split; ++r) sum[sub][0] += ld_cluster_f32(map_to_cta(at, r));
          }
          lin_finish<1, FORM == FORM_GATED>(p.q, sum[0], sum[1], b0, b1, (j0 + col) * p.q.ldo + i, (j0 + col) * p.q.ldp + i, 1);
        }
      }
    }
  }

  // ------------------------------------------------------------ teardown
  if (*reinterpret_cast<volatile int*>(&abort_flag)) {
    // copies still in flight land before shared memory is released
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR || SPLIT) cluster_sync_all();  // shared memory and TMEM stay until every CTA is done
  if (!SPLIT && warp == 1) {
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
  int form, bn, split, stages;
};

static size_t stage_size(const LinPick& c) {
  return (c.form == FORM_PLAIN ? 1 : 2) * static_cast<size_t>(kSubBytes) + static_cast<size_t>(c.bn / (c.pair ? 2 : 1)) * 128;
}

// Variant for a product, from its sizes.
static LinPick pick_variant(const LinArgs& q, int sms) {
  LinPick c;
  memset(&c, 0, sizeof(c));
  const int64_t groups = q.mode == LIN_ROWS ? q.groups : 1;
  const int64_t avg = q.mode == LIN_ROWS ? ceil_div64(q.rows, groups < q.rows ? groups : q.rows) : q.J;
  c.form = q.gated ? FORM_GATED : FORM_PLAIN;
  c.split = 1;
  const bool b_mn = q.b_mn != 0;
  const int64_t many = q.mode == LIN_REDUCE ? q.groups : groups;
  // pair tiles of 256 features x 256 tokens once they fill half of the GPU
  const int64_t pair_tiles = many * ceil_div64(q.I, 256) * ceil_div64(avg, 256);
  if (avg > 128 && pair_tiles * 2 * 2 >= sms) {
    c.pair = true;
    c.bn = 256;
    if (!q.gated && many * ceil_div64(q.I, 512) * ceil_div64(avg, 256) * 2 >= sms) c.form = FORM_WIDE;
  } else {
    c.bn = avg <= 16 ? 16 : avg <= 32 ? 32 : avg <= 64 ? 64 : 128;
    if (b_mn && c.bn < 64) c.bn = 64;
    if (q.mode == LIN_DENSE && c.bn <= 64) {
      const int64_t tiles = ceil_div64(q.I, 128) * ceil_div64(q.J, c.bn), blocks = ceil_div64(q.K, kKBlock);
      while (c.split < 8 && tiles * c.split * 2 <= 2 * sms && blocks >= 4 * c.split * 2) c.split *= 2;
    }
  }
  return c;
}

template <bool PAIR, int FORM, int EPI, bool SPLIT>
static int launch_variant(const CUtensorMap& a, const CUtensorMap& b, const LinUmma& p, int ctas, size_t smem,
                          cudaStream_t stream) {
  auto kern = linear_umma_kernel<PAIR, FORM, EPI, SPLIT>;
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
  cudaLaunchConfig_t lc;
  memset(&lc, 0, sizeof(lc));
  lc.gridDim = dim3(static_cast<unsigned>(ctas));
  lc.blockDim = dim3(128 + 32 * EPI);
  lc.dynamicSmemBytes = smem;
  lc.stream = stream;
  cudaLaunchAttribute attr[1];
  if (PAIR || SPLIT) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = PAIR ? 2 : static_cast<unsigned>(p.split);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    lc.attrs = attr;
    lc.numAttrs = 1;
  }
  const cudaError_t e = cudaLaunchKernelEx(&lc, kern, a, b, p);
  count_launch();
  return launch_status(e);
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
      if (pair && c.bn < 128) c.bn = 128;
      if (!pair && c.bn > 128) c.bn = 128;
      if (c.form == FORM_WIDE && c.bn < 256) c.form = FORM_PLAIN;
      if (cfg->split_k) {
        c.split = cfg->split_k;
        if (c.split > 1 && c.bn > 64) c.bn = 64;
      } else if (pair || c.bn > 64) {
        c.split = 1;
      }
    }
  }
  const bool two = !c.pair;
  const size_t limit = (two ? kTwoCtas : kOneCta) - 1024;
  int stages = static_cast<int>(limit / stage_size(c));
  if (stages > kLinStages) stages = kLinStages;
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
  const int64_t ti = ceil_div64(q.I, p.feat), tj = q.mode == LIN_ROWS ? 1 : ceil_div64(q.J, c.bn);
  p.tiles_i = static_cast<int>(ti);
  p.tiles_j = static_cast<int>(tj);
  // the most tiles there can be: a group ends in at most one partial tile
  const int64_t busy = q.mode == LIN_ROWS ? (q.groups < q.rows ? q.groups : q.rows) : 0;
  const int64_t most = q.mode == LIN_ROWS ? (q.rows / c.bn + busy) * ti : ti * tj * (q.mode == LIN_REDUCE ? q.groups : 1);
  if (most > 0x7fffffffll / 8) return FTB_E_TOO_LARGE;
  p.band = 8;
  const int acc_cols = subs * c.bn;
  p.acc_slots = c.form == FORM_WIDE ? 2 : c.split > 1 || 2 * acc_cols > (two ? 256 : 512) ? 1 : 2;
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
  p.status = status ? status : fallback_status();
  if (!p.status) return FTB_E_CUDA;

  const CUtensorMapDataType dt = q.f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint32_t ones[3] = {1, 1, 1};
  CUtensorMap ma, mb;
  int rc;
  if (q.mode == LIN_REDUCE) {
    // both operands are fetched row by row: 64 columns of four places per copy
    const uint32_t box[2] = {64, 1};
    const uint64_t da[2] = {static_cast<uint64_t>(q.I), static_cast<uint64_t>(q.gather_div ? q.src_rows : q.rows)};
    const uint64_t db[2] = {static_cast<uint64_t>(q.J), static_cast<uint64_t>(q.rows)};
    const uint64_t sa[1] = {static_cast<uint64_t>(q.lda) * 2}, sb[1] = {static_cast<uint64_t>(q.ldb) * 2};
    rc = make_tmap(&ma, dt, 2, q.a, da, sa, box, ones);
    if (!rc) rc = make_tmap(&mb, dt, 2, q.b, db, sb, box, ones);
    if (rc) return rc;
    p.oob_a = static_cast<int>(da[1]);
    p.oob_b = static_cast<int>(db[1]);
  } else {
    const uint64_t a_rows = static_cast<uint64_t>(q.gated ? 2 * q.I : q.I);
    const uint64_t a_groups = static_cast<uint64_t>(q.mode == LIN_ROWS ? q.groups : 1);
    uint64_t d[3] = {static_cast<uint64_t>(q.K), a_rows, a_groups};
    uint32_t box[3] = {64, 128, 1};
    if (q.a_mn) {
      d[0] = a_rows;
      d[1] = static_cast<uint64_t>(q.K);
      box[1] = 64;
    }
    const uint64_t sa[2] = {static_cast<uint64_t>(q.lda) * 2, d[1] * static_cast<uint64_t>(q.lda) * 2};
    rc = make_tmap(&ma, dt, 3, q.a, d, sa, box, ones);
    if (rc) return rc;
    const uint64_t b_rows = static_cast<uint64_t>(q.mode == LIN_ROWS ? (q.gather_div ? q.src_rows : q.rows) : q.J);
    if (q.gather_div) {
      const uint64_t db[2] = {static_cast<uint64_t>(q.K), b_rows};
      const uint64_t sb[1] = {static_cast<uint64_t>(q.ldb) * 2};
      const uint32_t gbox[2] = {64, 1};
      rc = make_tmap(&mb, dt, 2, q.b, db, sb, gbox, ones);
      p.oob_b = static_cast<int>(b_rows);
    } else {
      uint64_t db[3] = {static_cast<uint64_t>(q.K), b_rows, 1};
      uint32_t bbox[3] = {64, static_cast<uint32_t>(p.bj), 1};
      if (q.b_mn) {
        db[0] = b_rows;
        db[1] = static_cast<uint64_t>(q.K);
        bbox[1] = 64;
      }
      const uint64_t sb[2] = {static_cast<uint64_t>(q.ldb) * 2, db[1] * static_cast<uint64_t>(q.ldb) * 2};
      rc = make_tmap(&mb, dt, 3, q.b, db, sb, bbox, ones);
    }
    if (rc) return rc;
  }

  size_t smem = static_cast<size_t>(stages) * stage_size(c) + 1024;
  // A pair holds tensor memory while its CTAs wait for each other.  No other kernel with tensor memory may share the SM
  // with it (each could wait for columns that the other holds), so it always asks for most of the shared memory.
  if (c.pair && smem < 176 * 1024) smem = 176 * 1024;
  if (c.split > 1) {
    const int ctas = static_cast<int>(most) * c.split;
    return c.form == FORM_GATED ? launch_variant<false, FORM_GATED, 4, true>(ma, mb, p, ctas, smem, stream)
                                : launch_variant<false, FORM_PLAIN, 4, true>(ma, mb, p, ctas, smem, stream);
  }
  if (c.pair) {
    const int64_t units = sms / 2 < most ? sms / 2 : most;
    const int ctas = static_cast<int>(units) * 2;
    if (c.form == FORM_GATED) return launch_variant<true, FORM_GATED, 8, false>(ma, mb, p, ctas, smem, stream);
    if (c.form == FORM_WIDE) return launch_variant<true, FORM_WIDE, 8, false>(ma, mb, p, ctas, smem, stream);
    return launch_variant<true, FORM_PLAIN, 8, false>(ma, mb, p, ctas, smem, stream);
  }
  const int ctas = static_cast<int>(2 * sms < most ? 2 * sms : most);
  return c.form == FORM_GATED ? launch_variant<false, FORM_GATED, 4, false>(ma, mb, p, ctas, smem, stream)
                              : launch_variant<false, FORM_PLAIN, 4, false>(ma, mb, p, ctas, smem, stream);
}

}  // namespace ftb
