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

// True on one lane of a converged warp. The loops that issue copies and MMAs run
// on all lanes, with only the instruction itself under elect(): their operands
// then stay in uniform registers. Issued from a one-lane branch instead, a
// k-block's four MMAs and commit took 449 clocks instead of 215.
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ int warp_index() { return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0); }

__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(wgtc::smem_addr(bar)) : "memory");
}

// ---- epilogue ----------------------------------------------------------------

// Where and how results are stored: alpha, beta as in BLAS (C is read only when
// beta != 0), in 32 bits, rounded once to C's type. Lane i of a warp holds column
// l0 + i of W rows of C (ldc apart), of which the first `valid` exist. What bounds
// the stores is the rate at which an SM writes to L2, about 28 bytes a clock
// (measured with stores alone; this code reaches about 20): exchanging values
// between lanes to store 16-bit results as pairs, half as many stores, gained
// nothing.
struct Out {
  void *C;
  int64_t ldc;
  float alpha, beta;
  int type;
};

template <class T>
__device__ __forceinline__ T round_to(float x);
template <>
__device__ __forceinline__ float round_to<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half round_to<__half>(float x) { return __float2half_rn(x); }

// One column a lane. `at`: the element of row 0 in this lane's column. (The
// pointers step by ldc: W addresses kept apart would not fit the registers.)
template <class T, int W>
__device__ __forceinline__ void store_single(const Out &o, int64_t at, bool in, int valid, const float *acc) {
  if (!in) return;
  T *p = static_cast<T *>(o.C) + at;
  const int64_t ldc = o.ldc;
  const float alpha = o.alpha, beta = o.beta;
  if (beta == 0.0f) {
    if (valid >= W) {
#pragma unroll
      for (int j = 0; j < W; j++, p += ldc) *p = round_to<T>(alpha * acc[j]);
    } else {
#pragma unroll
      for (int j = 0; j < W; j++, p += ldc)
        if (j < valid) *p = round_to<T>(alpha * acc[j]);
    }
    return;
  }
  // The old values of eight rows are loaded before any is written: one memory
  // round trip for them.
#pragma unroll
  for (int c = 0; c < W; c += 8) {
    T old[8], *r = p;
#pragma unroll
    for (int j = 0; j < 8; j++, r += ldc)
      if (c + j < valid) old[j] = *r;
#pragma unroll
    for (int j = 0; j < 8; j++, p += ldc)
      if (c + j < valid) *p = round_to<T>(fmaf(beta, (float)old[j], alpha * acc[c + j]));
  }
}

template <int W>
__device__ __forceinline__ void store_cols(const Out &o, int64_t at, bool in, int valid, const float *acc) {
  if (o.type == WG_TYPE_F32) store_single<float, W>(o, at, in, valid, acc);
  else if (o.type == WG_TYPE_BF16) store_single<__nv_bfloat16, W>(o, at, in, valid, acc);
  else store_single<__half, W>(o, at, in, valid, acc);
}

// Eight epilogue warps: warp w of them reads lane quarter w % 4 and its half
// w / 4 of the columns, CPT of them.
constexpr int EPI_WARPS = 8;

// sum[] (+)= CPT accumulator columns from TMEM address `taddr`, of which `valid`
// are used (16 at a time: the sums leave few registers).
template <int CPT>
__device__ __forceinline__ void drain(uint32_t taddr, int valid, bool first, float (&sum)[CPT]) {
#pragma unroll
  for (int c = 0; c < CPT; c += 16) {
    if (c < valid) {
      uint32_t r[16];
      wgtc::tmem_ld_32x32b_x16(taddr + (uint32_t)c, r);
      wgtc::tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; j++) sum[c + j] = first ? __uint_as_float(r[j]) : sum[c + j] + __uint_as_float(r[j]);
    }
  }
}

// Stores drained sums; FP32: C is float32 whatever o.type says.
template <int CPT, bool FP32>
__device__ __forceinline__ void store_sums(const Out &o, int64_t at, bool in, int valid, const float (&sum)[CPT]) {
#pragma unroll
  for (int c = 0; c < CPT; c += 16)
    if (c < valid) {
      if (FP32) store_single<float, 16>(o, at + (int64_t)c * o.ldc, in, valid - c, sum + c);
      else store_cols<16>(o, at + (int64_t)c * o.ldc, in, valid - c, sum + c);
    }
}

// Stores CPT accumulator columns straight from TMEM (`from` false: zeros instead).
template <int CPT>
__device__ __forceinline__ void store_acc(uint32_t taddr, bool from, const Out &o, int64_t at, bool in, int valid) {
  constexpr int W = CPT < 32 ? CPT : 32;
  static_assert(W == 16 || W == 32, "");
#pragma unroll 1
  for (int c = 0; c < CPT && c < valid; c += W) {
    uint32_t r[W];
    float f[W];
    if (from) {
      if constexpr (W == 32) wgtc::tmem_ld_32x32b_x32(taddr + (uint32_t)c, r);
      else wgtc::tmem_ld_32x32b_x16(taddr + (uint32_t)c, r);
      wgtc::tmem_ld_wait();
    }
#pragma unroll
    for (int j = 0; j < W; j++) f[j] = from ? __uint_as_float(r[j]) : 0.0f;
    store_cols<W>(o, at + (int64_t)c * o.ldc, in, valid - c, f);
  }
}

// ---- contraction split over a cluster --------------------------------------------
//
// P CTAs of a cluster share a tile, each with its part of the k-blocks; CTA 0
// adds the others' sums to its own, in the order of their parts, and stores.
// Their epilogue warps write them into its shared memory, [part][column][lane],
// when its warps have read the last tile's. The writes are asynchronous and count
// themselves on CTA 0's barrier as they land, so nobody has to make them visible
// (a release at cluster scope behind a warp's own stores took about a thousand clocks);
// CTA 0 acquires them by waiting at cluster scope. Its arrivals that give the place back
// release its warps' reads at cluster scope, the others' waits acquire them; that release
// is not free either (0.2 us of 8 for 4 x 512 x 4096 in 8 groups) and left out where no
// further tile can ask for the place.

struct Parts {
  float *buf;        // CTA 0: (P - 1) x BN x 128 sums
  uint64_t *full;    // CTA 0: the others' sums have arrived (one arrival and their bytes)
  uint64_t *empty;   // others: CTA 0's warps have read them (8 arrivals)
  uint32_t turn;     // exchanges so far
};

// Joins sum[] over the cluster; true on CTA 0, which then holds the total. A warp
// of CTA `rank` calls it with its columns' place (`col` of the tile, lane `row`)
// and the tile's number of columns; `first`: the one warp that announces the bytes;
// `more`: the cluster has tiles after this one. False with *ok = false when a wait gave up.
template <int P, int BN, int CPT>
__device__ __forceinline__ bool join_parts(Parts &x, uint32_t rank, int col, int row, int valid, int columns, bool first,
                                           bool more, float (&sum)[CPT], bool *ok) {
  const uint32_t turn = x.turn++;
  const int lane = threadIdx.x & 31;
  if (rank) {
    if (!__all_sync(0xffffffffu, wgtc::mbar_wait_bounded_cluster(x.empty, (turn & 1u) ^ 1u, WAIT_BUDGET))) {
      *ok = false;
      return false;
    }
    const uint32_t to = wgtc::mapa_shared(wgtc::smem_addr(x.buf + ((int)(rank - 1) * BN + col) * 128 + row), 0);
    const uint32_t bar = wgtc::mapa_shared(wgtc::smem_addr(x.full), 0);
#pragma unroll
    for (int j = 0; j < CPT; j++)
      if (j < valid)
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(to + 512u * j),
                     "r"(__float_as_uint(sum[j])), "r"(bar)
                     : "memory");
    return false;
  }
  if (first && lane == 0) wgtc::mbar_arrive_expect_tx(x.full, (uint32_t)((P - 1) * columns * BL * 4));
  if (!__all_sync(0xffffffffu, wgtc::mbar_wait_bounded_cluster(x.full, turn & 1u, WAIT_BUDGET))) {
    *ok = false;
    return false;
  }
#pragma unroll
  for (int r = 0; r < P - 1; r++) {
    const float *from = x.buf + (r * BN + col) * 128 + row;
#pragma unroll
    for (int j = 0; j < CPT; j++)
      if (j < valid) sum[j] += from[128 * j];
  }
  __syncwarp();
  if (more && lane > 0 && lane < P)
    wgtc::mbar_arrive_cluster(wgtc::mapa_shared(wgtc::smem_addr(x.empty), (uint32_t)lane));
  return true;
}

// A place in a ring of N stages, and the parity of the round it is in.
template <int N>
struct Ring {
  int s = 0;
  uint32_t round = 0;
  __device__ __forceinline__ void next() {
    if (++s == N) {
      s = 0;
      round ^= 1u;
    }
  }
};

// ---- CTA pairs -------------------------------------------------------------------
//
// CG CTAs (1 or 2) share a tile of CG * 128 lanes; CTA 0 of a pair leads: it
// issues the MMAs, and its barriers count both CTAs' bytes and both epilogues.

template <int CG>
__device__ __forceinline__ uint32_t pair_rank() {
  if constexpr (CG == 2) return wgtc::cluster_ctarank();
  else return 0;
}
// All threads of a cluster of N CTAs meet.
template <int N>
__device__ __forceinline__ void cluster_sync() {
  if constexpr (N > 1) wgtc::cluster_sync();
  else __syncthreads();
}
// One arrival on the leader's copy of `bar`, and the leader's wait for them. What they
// signal for a pair is that TMEM has been read: tcgen05.wait::ld returned and the
// tcgen05 fences order it, so the arrival is relaxed, at the scope of both CTAs (a release
// there waits for the warp's own stores, about a thousand clocks).
template <int CG>
__device__ __forceinline__ void leader_arrive(uint64_t *bar) {
  if constexpr (CG == 2)
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                     wgtc::mapa_shared(wgtc::smem_addr(bar), 0))
                 : "memory");
  else mbar_arrive(bar);
}
template <int CG>
__device__ __forceinline__ bool leader_wait(uint64_t *bar, uint32_t parity) {
  if constexpr (CG == 2) return wgtc::mbar_wait_bounded_cluster(bar, parity, WAIT_BUDGET);
  else return wgtc::mbar_wait_bounded(bar, parity, WAIT_BUDGET);
}
// `bar` of every CTA of the pair receives one arrival when the MMAs issued so far complete.
template <int CG>
__device__ __forceinline__ void commit(uint64_t *bar) {
  if constexpr (CG == 2) wgtc::mma_commit_pair(bar, 3);
  else wgtc::mma_commit(bar);
}
// Tile loads counted on the leader's barrier; `lead` is its shared::cluster
// address (leader_addr) for a pair.
template <int CG>
__device__ __forceinline__ uint32_t leader_addr(uint64_t *bar) {
  if constexpr (CG == 2) return wgtc::mapa_shared(wgtc::smem_addr(bar), 0);
  else return wgtc::smem_addr(bar);
}
template <int CG>
__device__ __forceinline__ void load_2d(void *dst, const CUtensorMap *map, uint64_t *bar, uint32_t lead, int c0, int c1) {
  if constexpr (CG == 2) wgtc::tma_load_2d_pair(dst, map, lead, c0, c1);
  else wgtc::tma_load_2d(dst, map, bar, c0, c1);
}
template <int CG>
__device__ __forceinline__ void load_3d(void *dst, const CUtensorMap *map, uint64_t *bar, uint32_t lead, int c0, int c1,
                                        int c2) {
  if constexpr (CG == 2) wgtc::tma_load_3d_pair(dst, map, lead, c0, c1, c2);
  else wgtc::tma_load_3d(dst, map, bar, c0, c1, c2);
}
template <int CG>
__device__ __forceinline__ void pair_tmem_alloc(uint32_t *slot, uint32_t cols) {
  if constexpr (CG == 2) {
    wgtc::tmem_alloc_pair(slot, cols);
    wgtc::tmem_relinquish_pair();
  } else {
    wgtc::tmem_alloc(slot, cols);
    wgtc::tmem_relinquish();
  }
}
template <int CG>
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t cols) {
  if constexpr (CG == 2) wgtc::tmem_dealloc_pair(taddr, cols);
  else wgtc::tmem_dealloc(taddr, cols);
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

// A matrix's elements and the offsets are read and written by their own types.
inline wg_status check_aligned(const char *name, const void *p, int type) {
  if ((uintptr_t)p & (type == WG_TYPE_F32 ? 3 : 1))
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "%s must be aligned to its elements.", name);
  return WG_OK;
}
inline wg_status check_offsets(const int *offsets) {
  if ((uintptr_t)offsets & 3) return wg_fail(WG_ERR_INVALID_ARGUMENT, "offsets must be aligned to its elements.");
  return WG_OK;
}
// Whether matrices `stride` elements apart lie one after the other.
inline bool apart(int64_t stride, int64_t rows, int64_t cols, int64_t ld) {
  return rows <= 0 || (__int128)stride >= (__int128)(rows - 1) * ld + cols;
}

// Launches a kernel over clusters of CG CTAs with programmatic stream
// serialization (the kernel calls wg_pdl_wait before it touches memory).
template <int CG, class... KArgs, class... Args>
cudaError_t launch(void (*kern)(KArgs...), unsigned grid, unsigned block, size_t smem, cudaStream_t s, Args &&...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<Args &&>(args)...);
}

}  // namespace wgg

// While it lives, this thread may make calls that set things up (a memory pool,
// a kernel's attributes, its loading) although a stream is being captured: none
// of them is work on that stream.
struct wg_capture_relaxed {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  wg_capture_relaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~wg_capture_relaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

// Runs `queue` (which queues work on d->stream); on a handle opened with
// WG_DEVICE_TIMING and with gpu_ms given, waits and reports its device time.
// Calls on one handle from several threads queue one after the other: a call's
// copies in the handle's temporary memory and the product that reads them must
// be neighbours on the stream, and the handle's events are one pair.
template <class F>
wg_status wg_timed(wg_device *d, float *gpu_ms, F queue) {
  wg_capture_relaxed relaxed;
  std::lock_guard<std::mutex> turn(d->queueing);
  if (!gpu_ms || !(d->flags & WG_DEVICE_TIMING)) return queue();
  WG_CUDA(cudaEventRecord(d->ev_start, d->stream));
  const wg_status st = queue();
  if (st != WG_OK) return st;
  WG_CUDA(cudaEventRecord(d->ev_stop, d->stream));
  WG_CUDA(cudaEventSynchronize(d->ev_stop));
  WG_CUDA(cudaEventElapsedTime(gpu_ms, d->ev_start, d->ev_stop));
  return WG_OK;
}
