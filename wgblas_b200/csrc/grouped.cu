// Matrix products grouped by expert, 16-bit operands (bf16 or fp16), 32-bit
// accumulation on the tensor cores: wg_gemm_grouped_dev and wg_gemm_grouped_inner_dev of
// the C ABI. No counterpart in the reference; they stand beside its gemm for
// layers whose rows are routed to one of several weight matrices.
//
//   rows form:   C[r] = alpha * A[r] op(B_g) + beta * C[r]     r in group g's rows
//   inner form:  C_g  = alpha * A[rows of g]^T B[rows of g] + beta * C_g
//
// One persistent kernel: each CTA walks 128-lane x BN-column tiles (frame and
// numbering: grouped_common.cuh). Warp 0 streams 64-deep k-blocks of both
// operands into a ring (TMA, 128-byte swizzle), warp 1 issues tcgen05.mma into
// one of two TMEM accumulators, warps 2-5 store the other one.
#include <algorithm>
#include <cstring>

#include "grouped_common.cuh"

namespace {

using wgg::BL;
using wgg::mbar_arrive;
using wgg::WAIT_BUDGET;

constexpr int BK = 64;          // k-block: 64 16-bit elements, one 128-byte swizzle span
constexpr int EPI_WARPS = 4;
constexpr int LOAD_WARPS = 4;   // of the form that loads with plain loads
constexpr int CHUNK = 8192;     // bytes of 64 lines of one k-block
constexpr size_t SMEM_LIMIT = 227 * 1024;

// How the operands' storage gives the k-blocks (a "line" is 64 neighbouring
// elements, 128 bytes of shared memory):
//   ROWS_T  L side K-major (weights n x k), N side K-major (rows of A)
//   ROWS_N  L side MN-major (weights k x n), N side K-major
//   INNER   both MN-major (rows of A and of B are the contraction)
enum { ROWS_T = 0, ROWS_N = 1, INNER = 2 };

template <int BN_>
struct Shape {
  static constexpr int BN = BN_;
  static constexpr int L_BYTES = BL * 128;
  static constexpr int N_BYTES = BN * 128;
  static constexpr int STAGE = L_BYTES + N_BYTES;
  static constexpr int ACC_COLS = BN < 32 ? 32 : BN;
  static constexpr int MAX_STAGES = 10;
  // Ring depth: what shared memory holds beside the groups' tables.
  static constexpr int STAGES = (int)((SMEM_LIMIT - 12 * 1024) / STAGE) < MAX_STAGES
                                    ? (int)((SMEM_LIMIT - 12 * 1024) / STAGE)
                                    : MAX_STAGES;
  static constexpr size_t smem(int groups) {
    return 1024 + (size_t)STAGES * STAGE + 256 + 2 * ((size_t)groups + 1) * sizeof(int);
  }
};

struct Args {
  int groups;
  int rows;      // rows of the ragged operands
  int nl;        // extent of C's contiguous dimension
  int nn;        // inner form: rows of C
  int k;         // rows form: contraction length
  int tiles_l, tiles_n;
  const int *offsets;
  float alpha, beta;
  void *C;
  int64_t ldc, strideC;
  int ctype;
  uint32_t ab_format;  // idesc a/b format: 0 fp16, 1 bf16
  int l_group;         // 1: the L side's map has a group dimension (0: all groups share one matrix)
  // the operands for the plain-load form
  const uint16_t *L, *N;
  int64_t ldl, ldn, strideL;
  unsigned *dwords;
};

// Instruction descriptor of kind::f16, fp32 accumulation: c_format F32 (bits
// 4-5 = 1), a/b format (bits 7-9, 10-12), a/b MN-major (bits 15, 16), N>>3 at
// bits 17-22, M>>4 at bits 24-28.
__device__ __forceinline__ uint32_t idesc_f16(uint32_t fmt, int M, int N, bool a_mn, bool b_mn) {
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// Descriptor of an MN-major operand tile: 64-element (128-byte) chunks along
// MN, CHUNK bytes apart (leading byte offset), each with its k lines 128 bytes
// apart in groups of eight (stride byte offset 1024), 128-byte swizzle.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(CHUNK >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// One output tile: lanes [l0, l0 + 128) and columns [n0, n0 + nv) of group g,
// whose contraction (inner form) or rows (rows form) begin at row r0.
struct Tile {
  int g, l0, n0, nv;
  int r0;     // rows form: the tile's first row; inner form: the group's first row
  int kt;     // k-blocks
  int klen;   // contraction length
};

template <int MODE, class S>
__device__ __forceinline__ Tile tile_at(const Args &a, int64_t t, const int *start, const int *tile0) {
  Tile x;
  if (MODE == INNER) {
    const int per = a.tiles_l * a.tiles_n;
    x.g = (int)(t / per);
    const int local = (int)(t - (int64_t)x.g * per);
    const int tn = local % a.tiles_n;
    x.l0 = (local / a.tiles_n) * BL;
    x.n0 = tn * S::BN;
    x.nv = min(S::BN, a.nn - x.n0);
    x.r0 = start[x.g];
    x.klen = start[x.g + 1] - x.r0;
  } else {
    const int q = (int)(t / a.tiles_l);
    x.g = wgg::group_of(tile0, a.groups, q);
    const int ntok = tile0[x.g + 1] - tile0[x.g];
    const int local = (int)(t - (int64_t)tile0[x.g] * a.tiles_l);
    // The group's row tiles side by side, so that one tile of weights is read
    // by CTAs running at the same time.
    x.l0 = (local / ntok) * BL;
    const int first = (local % ntok) * S::BN;
    x.r0 = start[x.g] + first;
    x.n0 = first;
    x.nv = min(S::BN, start[x.g + 1] - x.r0);
    x.klen = a.k;
  }
  x.kt = a.alpha == 0.0f ? 0 : (x.klen + BK - 1) / BK;
  return x;
}

// Eight 16-bit elements at p, of which the first `valid` exist (the others are
// zero), by the widest loads p's alignment allows.
__device__ __forceinline__ uint4 load8(const uint16_t *p, int valid) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (valid <= 0) return v;
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  if (valid >= 8 && (at & 15) == 0) return __ldg(reinterpret_cast<const uint4 *>(p));
  uint32_t w[4] = {0, 0, 0, 0};
  if (valid >= 8 && (at & 3) == 0) {
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = __ldg(reinterpret_cast<const uint32_t *>(p) + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i < valid) w[i >> 1] |= (uint32_t)__ldg(p + i) << (16 * (i & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int MODE, class S, bool TMA>
__global__ void __launch_bounds__(TMA ? 192 : 320, 1)
grouped_kernel(const __grid_constant__ CUtensorMap map_l, const __grid_constant__ CUtensorMap map_n, const Args a) {
  constexpr bool L_MN = MODE != ROWS_T, N_MN = MODE == INNER;
  constexpr int STAGES = S::STAGES;
  constexpr int NBOX = S::BN < 64 ? S::BN : 64;  // rows of one N-side box
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = wgtc::smem_addr(smem_raw);
  uint8_t *smem = smem_raw + ((1024 - (base & 1023)) & 1023);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + (size_t)STAGES * S::STAGE);
  uint64_t *empty = full + STAGES;
  uint64_t *acc_full = empty + STAGES;  // [2]
  uint64_t *acc_empty = acc_full + 2;   // [2]
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  int *start = reinterpret_cast<int *>(smem + (size_t)STAGES * S::STAGE + 256);
  int *tile0 = start + a.groups + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      wgtc::mbar_init(&full[s], TMA ? 1 : 32 * LOAD_WARPS);
      wgtc::mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      wgtc::mbar_init(&acc_full[b], 1);
      wgtc::mbar_init(&acc_empty[b], 32 * EPI_WARPS);
    }
    *abort_flag = 0;
    wgtc::fence_barrier_init();
  }
  if (TMA && warp == 0 && lane == 0) {
    wgtc::prefetch_tensormap(&map_l);
    wgtc::prefetch_tensormap(&map_n);
  }
  if (warp == 1) {
    wgtc::tmem_alloc(tmem_slot, 2 * S::ACC_COLS);
    wgtc::tmem_relinquish();
  }
  wg_pdl_wait();
  wg_pdl_trigger();
  wgg::plan_groups(a.offsets, a.groups, a.rows, S::BN, start, MODE == INNER ? nullptr : tile0, nullptr, a.dwords);
  wgtc::tc_fence_before();
  __syncthreads();
  wgtc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int64_t tiles = MODE == INNER ? (int64_t)a.groups * a.tiles_l * a.tiles_n
                                      : (int64_t)tile0[a.groups] * a.tiles_l;

  if (TMA && warp == 0 && lane == 0) {
    // ---- TMA producer ----
    int64_t it = 0;
    bool ok = true;
    for (int64_t t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const Tile x = tile_at<MODE, S>(a, t, start, tile0);
      const int boxes = (x.nv + NBOX - 1) / NBOX;
      const uint32_t bytes = (uint32_t)(S::L_BYTES + boxes * NBOX * 128);
      for (int kb = 0; kb < x.kt; kb++, it++) {
        const int s = (int)(it % STAGES);
        const uint32_t ph = (uint32_t)(it / STAGES) & 1u;
        if (!wgtc::mbar_wait_bounded(&empty[s], ph ^ 1u, WAIT_BUDGET) || *abort_flag) {
          atomicOr(a.dwords + WG_DW_ERROR, WG_DERR_TMA_WAIT);
          *abort_flag = 1;
          ok = false;
          break;
        }
        uint8_t *st = smem + (size_t)s * S::STAGE;
        wgtc::mbar_arrive_expect_tx(&full[s], bytes);
        const int k0 = kb * BK;
        if (MODE == ROWS_T) {
          wgtc::tma_load_3d(st, &map_l, &full[s], k0, x.l0, x.g * a.l_group);
        } else if (MODE == ROWS_N) {
          wgtc::tma_load_3d(st, &map_l, &full[s], x.l0, k0, x.g * a.l_group);
          wgtc::tma_load_3d(st + CHUNK, &map_l, &full[s], x.l0 + 64, k0, x.g * a.l_group);
        } else {
          wgtc::tma_load_2d(st, &map_l, &full[s], x.l0, x.r0 + k0);
          wgtc::tma_load_2d(st + CHUNK, &map_l, &full[s], x.l0 + 64, x.r0 + k0);
        }
        uint8_t *sn = st + S::L_BYTES;
        for (int b = 0; b < boxes; b++) {
          if (N_MN) wgtc::tma_load_2d(sn + b * CHUNK, &map_n, &full[s], x.n0 + b * 64, x.r0 + k0);
          else wgtc::tma_load_2d(sn + b * NBOX * 128, &map_n, &full[s], k0, x.r0 + b * NBOX);
        }
      }
    }
    // Let every copy this thread issued land before the CTA can exit.
    for (int64_t q = it - STAGES > 0 ? it - STAGES : 0; q < it; q++)
      wgtc::mbar_wait_bounded(&full[q % STAGES], (uint32_t)(q / STAGES) & 1u, WAIT_BUDGET);
  } else if (!TMA && warp >= 6) {
    // ---- plain-load producer: four warps fill the same swizzled layout, zeros
    // outside the operands; any alignment ----
    const int tid = threadIdx.x - 192;
    int64_t it = 0;
    bool ok = true;
    for (int64_t t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const Tile x = tile_at<MODE, S>(a, t, start, tile0);
      const int nmma = (x.nv + 15) & ~15;
      const uint16_t *Lg = a.L + (int64_t)x.g * a.strideL;
      for (int kb = 0; kb < x.kt; kb++, it++) {
        const int s = (int)(it % STAGES);
        const uint32_t ph = (uint32_t)(it / STAGES) & 1u;
        ok = wgtc::mbar_wait_bounded(&empty[s], ph ^ 1u, WAIT_BUDGET) && *abort_flag == 0;
        if (!ok) {
          atomicOr(a.dwords + WG_DW_ERROR, WG_DERR_TMA_WAIT);
          *abort_flag = 1;
          break;
        }
        uint8_t *st = smem + (size_t)s * S::STAGE;
        const int k0 = kb * BK, kleft = x.klen - k0;
        const int nlines = N_MN ? 64 * ((nmma + 63) / 64) : nmma;
        const int units = (BL + nlines) * 8;
#pragma unroll 4
        for (int u = tid; u < units; u += 32 * LOAD_WARPS) {
          const int line = u >> 3, c = u & 7;
          const uint16_t *p;
          int valid;
          uint32_t dst;
          if (line < BL) {
            if (MODE == ROWS_T) {  // weight row l0 + line, columns k0 ..
              valid = x.l0 + line < a.nl ? kleft - c * 8 : 0;
              p = Lg + (int64_t)(x.l0 + line) * a.ldl + k0 + c * 8;
              dst = line * 128 + ((c ^ (line & 7)) << 4);
            } else {  // k line kk, columns l0 + 64 * chunk ..
              const int kk = line & 63, q = line >> 6, col = x.l0 + q * 64 + c * 8;
              valid = kk < kleft ? a.nl - col : 0;
              p = (MODE == INNER ? a.L + (int64_t)(x.r0 + k0 + kk) * a.ldl : Lg + (int64_t)(k0 + kk) * a.ldl) + col;
              dst = q * CHUNK + kk * 128 + ((c ^ (kk & 7)) << 4);
            }
          } else {
            const int l = line - BL;
            if (N_MN) {
              const int kk = l & 63, q = l >> 6, col = x.n0 + q * 64 + c * 8;
              valid = kk < kleft ? a.nn - col : 0;
              p = a.N + (int64_t)(x.r0 + k0 + kk) * a.ldn + col;
              dst = S::L_BYTES + q * CHUNK + kk * 128 + ((c ^ (kk & 7)) << 4);
            } else {
              valid = l < x.nv ? kleft - c * 8 : 0;
              p = a.N + (int64_t)(x.r0 + l) * a.ldn + k0 + c * 8;
              dst = S::L_BYTES + l * 128 + ((c ^ (l & 7)) << 4);
            }
          }
          *reinterpret_cast<uint4 *>(st + dst) = load8(p, valid);
        }
        wgtc::fence_proxy_async_smem();
        mbar_arrive(&full[s]);
      }
    }
  } else if (warp == 1) {
    // ---- MMA issuer (the whole warp, for the zero rows of a ragged end; lane 0 issues) ----
    int64_t it = 0;
    int used = 0;
    bool ok = true;
    for (int64_t t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const Tile x = tile_at<MODE, S>(a, t, start, tile0);
      if (x.kt == 0) continue;
      const int nmma = (x.nv + 15) & ~15;
      const uint32_t idesc = idesc_f16(a.ab_format, BL, nmma, L_MN, N_MN);
      const int b = used & 1;
      ok = wgtc::mbar_wait_bounded(&acc_empty[b], ((uint32_t)(used >> 1) & 1u) ^ 1u, WAIT_BUDGET) && *abort_flag == 0;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        if (lane == 0) atomicOr(a.dwords + WG_DW_ERROR, WG_DERR_MMA_WAIT);
        *abort_flag = 1;
        break;
      }
      wgtc::tc_fence_after();
      const uint32_t d_tmem = tmem + (uint32_t)(b * S::ACC_COLS);
      for (int kb = 0; kb < x.kt; kb++, it++) {
        const int s = (int)(it % STAGES);
        ok = wgtc::mbar_wait_bounded(&full[s], (uint32_t)(it / STAGES) & 1u, WAIT_BUDGET) && *abort_flag == 0;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          if (lane == 0) atomicOr(a.dwords + WG_DW_ERROR, WG_DERR_TMA_WAIT);
          *abort_flag = 1;
          break;
        }
        uint8_t *st = smem + (size_t)s * S::STAGE;
        const int left = min(BK, x.klen - kb * BK);
        const int steps = (left + 15) >> 4;
        if (TMA && MODE == INNER && (left & 15)) {
          // The lines past the group's last row hold the next group's (whatever
          // they are, infinities among them): zero those the last MMA would read.
          const int lines = steps * 16 - left, chunks = 2 + (nmma + 63) / 64;
          for (int u = lane; u < chunks * lines * 8; u += 32) {
            const int c = u & 7, r = (u >> 3) % lines, q = (u >> 3) / lines;
            *reinterpret_cast<uint4 *>(st + q * CHUNK + (left + r) * 128 + c * 16) = make_uint4(0, 0, 0, 0);
          }
          wgtc::fence_proxy_async_smem();
          __syncwarp();
        }
        wgtc::tc_fence_after();
        if (lane == 0) {
          const uint32_t sl = wgtc::smem_addr(st), sn = sl + S::L_BYTES;
          for (int kk = 0; kk < steps; kk++) {
            const uint64_t dl = L_MN ? smem_desc_mn(sl + kk * 2048) : wgtc::smem_desc_kmajor(sl + kk * 32, 128);
            const uint64_t dn = N_MN ? smem_desc_mn(sn + kk * 2048) : wgtc::smem_desc_kmajor(sn + kk * 32, 128);
            mma_f16(d_tmem, dl, dn, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
          }
          wgtc::mma_commit(&empty[s]);
        }
        __syncwarp();
      }
      if (!ok) break;
      if (lane == 0) wgtc::mma_commit(&acc_full[b]);
      used++;
    }
  } else if (warp >= 2 && warp < 2 + EPI_WARPS) {
    // ---- epilogue ----
    const int q = warp & 3;
    int used = 0;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
      const Tile x = tile_at<MODE, S>(a, t, start, tile0);
      const int b = used & 1;
      bool ready = true;
      if (x.kt) {
        ready = wgtc::mbar_wait_bounded(&acc_full[b], (uint32_t)(used >> 1) & 1u, WAIT_BUDGET) && *abort_flag == 0;
        ready = __all_sync(0xffffffffu, ready);
        if (!ready) {
          if (lane == 0) atomicOr(a.dwords + WG_DW_ERROR, WG_DERR_MMA_WAIT);
          *abort_flag = 1;
          break;
        }
        wgtc::tc_fence_after();
      }
      const int l = x.l0 + q * 32 + lane;
      const int64_t row = MODE == INNER ? x.n0 : x.r0;
      const int64_t at = (MODE == INNER ? (int64_t)x.g * a.strideC : 0) + row * a.ldc + l;
      const uint32_t trow = tmem + (uint32_t)(b * S::ACC_COLS) + ((uint32_t)(q * 32) << 16);
      for (int c = 0; c < x.nv; c += 32) {
        uint32_t r[32];
        if (x.kt) {
          wgtc::tmem_ld_32x32b_x32(trow + (uint32_t)c, r);
          wgtc::tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; j++) r[j] = 0;
        }
        if (l < a.nl) wgg::store_cols<32>(a.C, a.ctype, at + (int64_t)c * a.ldc, a.ldc, x.nv - c, a.alpha, a.beta, r);
      }
      if (x.kt) {
        wgtc::tc_fence_before();
        mbar_arrive(&acc_empty[b]);
        used++;
      }
    }
  }

  wgtc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    wgtc::tc_fence_after();
    wgtc::tmem_dealloc(tmem, 2 * S::ACC_COLS);
  }
}

// ---- host side ------------------------------------------------------------

bool encode(CUtensorMap *map, int type, const void *ptr, int rank, const cuuint64_t *dims, const cuuint64_t *strides,
            const cuuint32_t *box) {
  wg_encode_tiled_fn fn = wg_encode_tiled();
  if (!fn) return false;
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapDataType dt = type == WG_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return fn(map, dt, rank, const_cast<void *>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A TMA map can read a row-major matrix whose base and row length are whole
// 16-byte units (cuTensorMapEncodeTiled's rule; strides below 2^40 bytes).
bool mappable(const void *p, int64_t ld) {
  return ((uintptr_t)p & 15) == 0 && (ld * 2) % 16 == 0 && ld * 2 < ((int64_t)1 << 40);
}

template <int MODE, class S>
wg_status launch(wg_device *d, const char *family, Args &a, int type, int64_t row_tiles_most) {
  const bool l_rows = MODE != INNER;
  // Weights shared by all groups (stride 0, or one group) need no group dimension.
  a.l_group = l_rows && a.groups > 1 && a.strideL != 0;
  bool tma = mappable(a.L, a.ldl) && mappable(a.N, a.ldn) &&
             (!a.l_group || ((a.strideL * 2) % 16 == 0 && a.strideL * 2 < ((int64_t)1 << 40)));
  CUtensorMap ml, mn;
  memset(&ml, 0, sizeof ml);
  memset(&mn, 0, sizeof mn);
  if (tma) {
    const cuuint64_t ldl = (cuuint64_t)a.ldl * 2, ldn = (cuuint64_t)a.ldn * 2;
    if (MODE == INNER) {
      const cuuint64_t dl[2] = {(cuuint64_t)a.nl, (cuuint64_t)a.rows}, dn[2] = {(cuuint64_t)a.nn, (cuuint64_t)a.rows};
      const cuuint32_t box[2] = {64, 64};
      tma = encode(&ml, type, a.L, 2, dl, &ldl, box) && encode(&mn, type, a.N, 2, dn, &ldn, box);
    } else {
      const int64_t lrows = MODE == ROWS_T ? a.nl : a.k, lcols = MODE == ROWS_T ? a.k : a.nl;
      const cuuint64_t dl[3] = {(cuuint64_t)lcols, (cuuint64_t)lrows, a.l_group ? (cuuint64_t)a.groups : 1};
      const cuuint64_t sl[2] = {ldl, a.l_group ? (cuuint64_t)a.strideL * 2 : ldl * (cuuint64_t)lrows};
      const cuuint32_t bl[3] = {64, MODE == ROWS_T ? (cuuint32_t)BL : 64u, 1};
      const cuuint64_t dn[2] = {(cuuint64_t)a.k, (cuuint64_t)a.rows};
      const cuuint32_t bn[2] = {64, (cuuint32_t)std::min(S::BN, 64)};
      tma = encode(&ml, type, a.L, 3, dl, sl, bl) && encode(&mn, type, a.N, 2, dn, &ldn, bn);
    }
  }
  const size_t smem = S::smem(a.groups);
  const int64_t most = row_tiles_most * a.tiles_l;
  const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(most, d->sm_count));
  wg_launch_scope scope(d, family);
  if (tma) {
    WG_CUDA(wg_kernel_smem(grouped_kernel<MODE, S, true>, SMEM_LIMIT));
    WG_CUDA(wg_launch_pdl(grouped_kernel<MODE, S, true>, dim3(grid), dim3(192), smem, d->stream, ml, mn, a));
  } else {
    WG_CUDA(wg_kernel_smem(grouped_kernel<MODE, S, false>, SMEM_LIMIT));
    WG_CUDA(wg_launch_pdl(grouped_kernel<MODE, S, false>, dim3(grid), dim3(320), smem, d->stream, ml, mn, a));
  }
  WG_CUDA(cudaGetLastError());
  return WG_OK;
}

// Columns of a tile: enough for a group's rows when they are spread evenly, as
// few as its rows fill otherwise.
template <int MODE>
wg_status launch_rows(wg_device *d, Args &a, int type) {
  const int64_t avg = (a.rows + a.groups - 1) / a.groups;
  if (avg <= 32) return launch<MODE, Shape<32>>(d, "gemm_grouped", a, type, a.rows / 32 + a.groups);
  if (avg <= 64) return launch<MODE, Shape<64>>(d, "gemm_grouped", a, type, a.rows / 64 + a.groups);
  if (avg <= 128) return launch<MODE, Shape<128>>(d, "gemm_grouped", a, type, a.rows / 128 + a.groups);
  return launch<MODE, Shape<256>>(d, "gemm_grouped", a, type, a.rows / 256 + a.groups);
}

wg_status launch_inner(wg_device *d, Args &a, int type) {
  a.tiles_n = (a.nn + 255) / 256;
  if (a.nn <= 128) {
    a.tiles_n = (a.nn + 127) / 128;
    return launch<INNER, Shape<128>>(d, "gemm_grouped_inner", a, type, (int64_t)a.groups * a.tiles_n);
  }
  return launch<INNER, Shape<256>>(d, "gemm_grouped_inner", a, type, (int64_t)a.groups * a.tiles_n);
}

constexpr int64_t LIM = (int64_t)1 << 31;

wg_status check_common(const wg_device *d, int type, int ctype, int64_t groups, int64_t m, int64_t n, int64_t k) {
  if (!d) return wg_fail(WG_ERR_INVALID_ARGUMENT, "device is NULL");
  if (type != WG_TYPE_BF16 && type != WG_TYPE_F16)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "A and B must be bfloat16 or float16.");
  if (ctype != WG_TYPE_F32 && ctype != type)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "C must have the type of A and B, or float32.");
  if (groups < 0 || m < 0 || n < 0 || k < 0)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "groups, m, n, and k must be non-negative.");
  if (groups > WG_MAX_GROUPS)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "groups must be at most %d.", WG_MAX_GROUPS);
  // Row and column numbers are 32-bit in the kernels and their copies, with room for one tile.
  if (m >= LIM - 1024 || n >= LIM - 1024 || k >= LIM - 1024)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "dimensions must be below 2^31 - 1024");
  return WG_OK;
}

wg_status check_ld(const char *name, int64_t ld, int64_t cols) {
  if (ld <= 0) return wg_fail(WG_ERR_INVALID_ARGUMENT, "lda, ldb, and ldc must be positive.");
  if (ld < cols) return wg_fail(WG_ERR_INVALID_ARGUMENT, "%s must be >= cols of its matrix as stored.", name);
  if (ld >= ((int64_t)1 << 40)) return wg_fail(WG_ERR_INVALID_ARGUMENT, "leading dimensions must be below 2^40");
  return WG_OK;
}

}  // namespace

extern "C" wg_status wg_gemm_grouped_dev(wg_device *d, int type, int ctype, int transB, int64_t groups, int64_t m,
                                     int64_t n, int64_t k, float alpha, const void *A, int64_t lda, const void *B,
                                     int64_t ldb, int64_t strideB, const int *offsets, float beta, void *C,
                                     int64_t ldc, float *gpu_ms) {
  if (gpu_ms) *gpu_ms = 0.0f;
  wg_status st = check_common(d, type, ctype, groups, m, n, k);
  if (st != WG_OK) return st;
  if (transB != 0 && transB != 1)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "transB must be 'no-transpose' or 'transpose'.");
  if ((st = check_ld("lda", lda, k)) != WG_OK || (st = check_ld("ldb", ldb, transB ? k : n)) != WG_OK ||
      (st = check_ld("ldc", ldc, n)) != WG_OK)
    return st;
  if (strideB < 0 || strideB >= ((int64_t)1 << 40))
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "strideB must be non-negative and below 2^40.");
  if (groups == 0 || m == 0 || n == 0) return WG_OK;
  if (!offsets || !C || (k > 0 && alpha != 0.0f && (!A || !B)))
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "operand pointer is NULL");
  st = wgg::check_arch(d);
  if (st != WG_OK) return st;
  if (beta == 1.0f && (alpha == 0.0f || k == 0)) return WG_OK;  // C stays as it is
  wg_device_guard guard(d->ordinal);
  Args a = {};
  a.groups = (int)groups;
  a.rows = (int)m;
  a.nl = (int)n;
  a.k = (int)k;
  a.tiles_l = (int)((n + BL - 1) / BL);
  a.offsets = offsets;
  a.alpha = k > 0 ? alpha : 0.0f;
  a.beta = beta;
  a.C = C;
  a.ldc = ldc;
  a.ctype = ctype;
  a.ab_format = type == WG_TYPE_BF16 ? 1u : 0u;
  a.L = static_cast<const uint16_t *>(B);
  a.ldl = ldb;
  a.strideL = strideB;
  a.N = static_cast<const uint16_t *>(A);
  a.ldn = lda;
  a.dwords = d->dwords;
  return wg_timed(d, gpu_ms, [&] { return transB ? launch_rows<ROWS_T>(d, a, type) : launch_rows<ROWS_N>(d, a, type); });
}

extern "C" wg_status wg_gemm_grouped_inner_dev(wg_device *d, int type, int ctype, int64_t groups, int64_t m, int64_t n,
                                           int64_t k, float alpha, const void *A, int64_t lda, const void *B,
                                           int64_t ldb, const int *offsets, float beta, void *C, int64_t ldc,
                                           int64_t strideC, float *gpu_ms) {
  if (gpu_ms) *gpu_ms = 0.0f;
  wg_status st = check_common(d, type, ctype, groups, m, n, k);
  if (st != WG_OK) return st;
  if ((st = check_ld("lda", lda, m)) != WG_OK || (st = check_ld("ldb", ldb, n)) != WG_OK ||
      (st = check_ld("ldc", ldc, n)) != WG_OK)
    return st;
  // Each group writes its own matrix.
  if (groups > 1 && (strideC < (m > 0 ? (m - 1) * ldc + n : 0) || strideC >= ((int64_t)1 << 40)))
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "strideC must be at least one matrix of C and below 2^40.");
  if (groups == 0 || m == 0 || n == 0) return WG_OK;
  if (!offsets || !C || (k > 0 && alpha != 0.0f && (!A || !B)))
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "operand pointer is NULL");
  st = wgg::check_arch(d);
  if (st != WG_OK) return st;
  if (beta == 1.0f && (alpha == 0.0f || k == 0)) return WG_OK;  // C stays as it is
  wg_device_guard guard(d->ordinal);
  Args a = {};
  a.groups = (int)groups;
  a.rows = (int)k;
  a.nl = (int)n;
  a.nn = (int)m;
  a.tiles_l = (int)((n + BL - 1) / BL);
  a.offsets = offsets;
  a.alpha = k > 0 ? alpha : 0.0f;
  a.beta = beta;
  a.C = C;
  a.ldc = ldc;
  a.strideC = groups > 1 ? strideC : 0;
  a.ctype = ctype;
  a.ab_format = type == WG_TYPE_BF16 ? 1u : 0u;
  a.L = static_cast<const uint16_t *>(B);
  a.ldl = ldb;
  a.N = static_cast<const uint16_t *>(A);
  a.ldn = lda;
  a.dwords = d->dwords;
  return wg_timed(d, gpu_ms, [&] { return launch_inner(d, a, type); });
}
