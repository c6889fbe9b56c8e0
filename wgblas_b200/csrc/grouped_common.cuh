// Pieces shared by the products whose rows are grouped by expert (grouped.cu:
// 16-bit operands; mx.cu: MXFP4 operands): reading the row ranges of the groups
// on the device, numbering the output tiles over them, and the epilogue's
// stores.
//
// Frame. C is row-major. Its contiguous dimension lies along the TMEM lanes
// (the "L side": an expert's weight rows or columns), its rows along the
// accumulator's columns (the "N side": a group's rows). So a thread holds one
// column of C for many rows, and a warp's store of one row is 32 neighbouring
// elements whatever C's leading dimension is; a tile that ends inside a group
// only shortens the loop over rows.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "internal.h"
#include "tcgen05.cuh"

namespace wgg {

constexpr int BL = 128;                        // lanes of a tile
constexpr long long WAIT_BUDGET = 4000000000LL;  // SM clocks (~2 s) before a wait gives up

// ---- the groups' row ranges --------------------------------------------------

// start[g] .. start[g + 1] are group g's rows: the caller's offsets clamped to
// [0, rows] and made non-decreasing by a running maximum, so that no offset a
// caller can pass leads outside the operands or gives a row to two groups.
// Offsets this changes are reported in the device error word. tile0[g] (when
// given) is the number of `bn`-row tiles of the groups before g, atom0[g] (when
// given) the number of 128-row tiles before it. Without offsets there is one
// group, all rows. All threads of the block call
// it; the results are visible to all of them when it returns.
__device__ __forceinline__ void plan_groups(const int *offsets, int groups, int rows, int bn, int *start, int *tile0,
                                            int *atom0, unsigned *dwords) {
  for (int j = threadIdx.x; j <= groups; j += blockDim.x) start[j] = offsets ? offsets[j] : (j ? rows : 0);
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int top = 0;
    bool bad = false;
    for (int base = 0; base <= groups; base += 32) {
      const int j = base + lane;
      const int raw = j <= groups ? start[j] : 0;
      int v = max(min(raw, rows), 0);
      if (j > groups) v = 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v = max(v, o);
      }
      v = max(v, top);
      if (j <= groups) {
        start[j] = v;
        bad |= v != raw;
      }
      top = __shfl_sync(0xffffffffu, v, 31);
    }
    if (bad && blockIdx.x == 0) atomicOr(dwords + WG_DW_ERROR, WG_DERR_OFFSETS);
    __syncwarp();
    int tiles = 0, atoms = 0;
    if (tile0) {
      if (lane == 0) {
        tile0[0] = 0;
        if (atom0) atom0[0] = 0;
      }
      for (int base = 0; base < groups; base += 32) {
        const int j = base + lane;
        const int n = j < groups ? start[j + 1] - start[j] : 0;
        int t = (n + bn - 1) / bn, a = (n + 127) / 128;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int ot = __shfl_up_sync(0xffffffffu, t, d), oa = __shfl_up_sync(0xffffffffu, a, d);
          if (lane >= d) {
            t += ot;
            a += oa;
          }
        }
        t += tiles;
        a += atoms;
        if (j < groups) {
          tile0[j + 1] = t;
          if (atom0) atom0[j + 1] = a;
        }
        tiles = __shfl_sync(0xffffffffu, t, 31);
        atoms = __shfl_sync(0xffffffffu, a, 31);
      }
    }
  }
  __syncthreads();
}

// The group whose tiles contain row tile q: the last g with tile0[g] <= q
// (groups without rows have tile0[g] == tile0[g + 1] and are passed over).
__device__ __forceinline__ int group_of(const int *tile0, int groups, int q) {
  int lo = 0, hi = groups;  // tile0[lo] <= q < tile0[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tile0[mid] <= q) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(wgtc::smem_addr(bar)) : "memory");
}

// ---- epilogue ----------------------------------------------------------------

// The element types of operands and results (WG_TYPE_* of the C ABI).
__device__ __forceinline__ float load_c(const void *c, int64_t i, int type) {
  if (type == WG_TYPE_F32) return static_cast<const float *>(c)[i];
  if (type == WG_TYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(c)[i]);
  return __half2float(static_cast<const __half *>(c)[i]);
}

// Stores W accumulator columns of one lane: row r0 + j of C (ldc apart), for
// j < valid. alpha, beta as in BLAS (C is read only when beta != 0), in 32
// bits, rounded once to C's type. `at` points at the lane's element of the
// first row.
template <class T, int W, class Round>
__device__ __forceinline__ void store_typed(T *at, int64_t ldc, int valid, float alpha, float beta,
                                            const uint32_t (&acc)[W], Round round) {
  if (beta == 0.0f) {
    if (valid >= W) {
#pragma unroll
      for (int j = 0; j < W; j++) at[j * ldc] = round(alpha * __uint_as_float(acc[j]));
    } else {
#pragma unroll
      for (int j = 0; j < W; j++)
        if (j < valid) at[j * ldc] = round(alpha * __uint_as_float(acc[j]));
    }
    return;
  }
  // The old values of a chunk are loaded before any is written: one memory
  // round trip for the chunk.
  T old[W];
#pragma unroll
  for (int j = 0; j < W; j++)
    if (j < valid) old[j] = at[j * ldc];
#pragma unroll
  for (int j = 0; j < W; j++)
    if (j < valid) at[j * ldc] = round(fmaf(beta, (float)old[j], alpha * __uint_as_float(acc[j])));
}

template <int W>
__device__ __forceinline__ void store_cols(void *C, int type, int64_t at, int64_t ldc, int valid, float alpha,
                                           float beta, const uint32_t (&acc)[W]) {
  if (type == WG_TYPE_BF16)
    store_typed<__nv_bfloat16, W>(static_cast<__nv_bfloat16 *>(C) + at, ldc, valid, alpha, beta, acc,
                                  [](float x) { return __float2bfloat16_rn(x); });
  else if (type == WG_TYPE_F16)
    store_typed<__half, W>(static_cast<__half *>(C) + at, ldc, valid, alpha, beta, acc,
                           [](float x) { return __float2half_rn(x); });
  else
    store_typed<float, W>(static_cast<float *>(C) + at, ldc, valid, alpha, beta, acc, [](float x) { return x; });
}

// ---- host side ------------------------------------------------------------

// Whether the device can run the sm_100a kernels in this library at all.
inline wg_status check_arch(const wg_device *d) {
  if (d->cc_major != 10)
    return wg_fail(WG_ERR_NOT_SUPPORTED,
                   "device %d (%s, sm_%d%d) is not a Blackwell sm_100 device; this library is built "
                   "for sm_100a only", d->ordinal, d->name, d->cc_major, d->cc_minor);
  return WG_OK;
}

}  // namespace wgg

// Runs `queue` (which queues work on d->stream); on a handle opened with
// WG_DEVICE_TIMING and with gpu_ms given, waits and reports its device time.
template <class F>
wg_status wg_timed(wg_device *d, float *gpu_ms, F queue) {
  if (!gpu_ms || !(d->flags & WG_DEVICE_TIMING)) return queue();
  WG_CUDA(cudaEventRecord(d->ev_start, d->stream));
  const wg_status st = queue();
  if (st != WG_OK) return st;
  WG_CUDA(cudaEventRecord(d->ev_stop, d->stream));
  WG_CUDA(cudaEventSynchronize(d->ev_stop));
  WG_CUDA(cudaEventElapsedTime(gpu_ms, d->ev_start, d->ev_stop));
  return WG_OK;
}
