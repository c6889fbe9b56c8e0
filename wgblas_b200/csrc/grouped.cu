// Matrix products grouped by expert, 16-bit operands (bf16 or fp16), 32-bit
// accumulation on the tensor cores: wg_gemm_grouped_dev and wg_gemm_grouped_inner_dev of
// the C ABI. No counterpart in the reference; they stand beside its gemm for
// layers whose rows are routed to one of several weight matrices.
//
//   rows form:   C[r] = alpha * A[r] op(B_g) + beta * C[r]     r in group g's rows
//   inner form:  C_g  = alpha * A[rows of g]^T B[rows of g] + beta * C_g
//
// One persistent kernel over 128-lane (256 for a CTA pair) x BN-column tiles
// (frame and numbering: grouped_common.cuh). Warp 0 streams 64-deep k-blocks of
// both operands into a ring (TMA, 128-byte swizzle), warp 1 issues tcgen05.mma
// into one of two TMEM accumulators, warps 2-9 add up and store the other one.
// Forms:
//   pairs, BN 256   compute-bound calls. A 128 x 256 tile on one CTA needs 96
//                   bytes of operands a clock from L2, more than an SM gets; a
//                   pair's 256 x 256 tile needs 64.
//   one CTA         calls with few rows a group, bound by the weights' bytes.
// Operands that a TMA map cannot describe (odd row lengths, unaligned bases) are
// first copied to aligned rows in a stream-ordered temporary.
#include <algorithm>
#include <cstring>

#include "grouped_common.cuh"

namespace {

using wgg::BL;
using wgg::mbar_arrive;
using wgg::WAIT_BUDGET;

constexpr int BK = 64;          // k-block: 64 16-bit elements, one 128-byte swizzle span
constexpr int EPI_WARPS = wgg::EPI_WARPS;
// The tensor core truncates when it adds to the accumulator: on data of one sign up to
// 5.9e-9 of the sum a contraction row (measured, fp16 and bf16 values spread over
// [0.5, 1.5]; normal data 1.2e-9). So accumulators are drained every so many k-blocks and
// the drained sums added in registers, rounded to nearest:
//   SEG   fp32 results (at most 2.4e-6 of a sum is lost to truncation), split contractions;
//   LONG  16-bit results: 8192 rows, 4.8e-5, a tenth of fp16's half step (2^-11). bf16's
//         (2^-8) is eight times that, so its sums are drained beyond 65536 rows only.
// (An fp16 weight gradient of 2048 x 4096 over 16384 rows in 8 groups takes 169 us so, 165
// from one accumulator.)
constexpr int SEG = 8, LONG = 128;
// Rows of a 16-bit result's contraction that one accumulator takes whole.
constexpr int whole_rows(int type) { return type == WG_TYPE_BF16 ? 8 * LONG * BK : LONG * BK; }
constexpr long long BLOCK_BUDGET = 5000;  // clocks a k-block may take (230 to 512 where nothing delays it)
constexpr int CHUNK = 8192;     // bytes of 64 lines of one k-block
constexpr size_t SMEM_LIMIT = 227 * 1024;

// How the operands' storage gives the k-blocks (a "line" is 64 neighbouring
// elements, 128 bytes of shared memory):
//   ROWS_T  L side K-major (weights n x k), N side K-major (rows of A)
//   ROWS_N  L side MN-major (weights k x n), N side K-major
//   INNER   both MN-major (rows of A and of B are the contraction)
enum { ROWS_T = 0, ROWS_N = 1, INNER = 2 };

// CG CTAs (a pair or one) share a tile's lanes, P CTAs its contraction.
template <int CG_, int BN_, int P_ = 1>
struct Shape {
  static constexpr int CG = CG_, BN = BN_, P = P_, CLUSTER = CG * P;
  static_assert(CG == 1 || P == 1, "a pair shares lanes or contraction, not both");
  static constexpr int TL = CG * BL;            // lanes of a tile
  static constexpr int CPT = BN / 2;            // accumulator columns of an epilogue thread
  static constexpr int L_BYTES = BL * 128;
  static constexpr int N_BYTES = BN / CG * 128;  // each CTA of a pair holds half of the columns' lines
  static constexpr int STAGE = L_BYTES + N_BYTES;
  static constexpr int PARTS = (P - 1) * BN * BL * 4;
  static constexpr int MAX_STAGES = 10;
  // Ring depth: what shared memory holds beside the groups' tables and the parts.
  static constexpr int FIT = (int)((SMEM_LIMIT - 26 * 1024 - PARTS) / STAGE);
  static constexpr int STAGES = FIT < MAX_STAGES ? FIT : MAX_STAGES;
  // Inner form: places for the last 16 lines of a group whose length is no
  // multiple of 16, beside the ring (see the kernel).
  static constexpr int ENDS = 2, END = (2 + (BN / CG + 63) / 64) * 2048;
  static constexpr int BARS = 2 * STAGES + 4 * ENDS + 6;
  static constexpr size_t ends = (size_t)STAGES * STAGE;
  static constexpr size_t parts = ends + (size_t)ENDS * END;
  static constexpr size_t bars = parts + PARTS;
  static constexpr size_t tables = bars + (BARS * 8 + 8 + 15) / 16 * 16;
  static constexpr size_t smem(int groups) { return 1024 + tables + 2 * ((size_t)groups + 1) * sizeof(int); }
  static constexpr int NMMA_STEP = CG * 16;
};

struct Args {
  int groups;
  int rows;      // rows of the ragged operands
  int nl;        // extent of C's contiguous dimension
  int nn;        // inner form: rows of C
  int k;         // rows form: contraction length
  int tiles_l, tiles_n;
  const int *offsets;
  wgg::Out out;
  int64_t strideC;
  uint32_t ab_format;  // idesc a/b format: 0 fp16, 1 bf16
  int l_group;         // 1: the L side's map has a group dimension (0: all groups share one matrix)
  // the operands
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
// MN, `chunk` bytes apart (leading byte offset), each with its k lines 128 bytes
// apart in groups of eight (stride byte offset 1024), 128-byte swizzle.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t saddr, int chunk = CHUNK) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(chunk >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// One output tile: lanes [l0, l0 + TL) and columns [n0, n0 + nv) of group g,
// whose contraction (inner form) or rows (rows form) begin at row r0.
struct Tile {
  int g, l0, n0, nv;
  int r0;     // rows form: the tile's first row; inner form: the group's first row
  int kt;     // k-blocks
  int klen;   // contraction length (inner form: without `end`)
  int k_lo, k_hi;  // this CTA's k-blocks
  int end;    // inner form: lines past the last whole 16, when this CTA takes them
  bool any;   // anything to contract
};

template <int MODE, class S>
__device__ __forceinline__ Tile tile_at(const Args &a, int64_t t, const int *start, const int *tile0, uint32_t rank) {
  Tile x;
  if (MODE == INNER) {
    const int per = a.tiles_l * a.tiles_n;
    x.g = (int)(t / per);
    const int local = (int)(t - (int64_t)x.g * per);
    const int tn = local % a.tiles_n;
    x.l0 = (local / a.tiles_n) * S::TL;
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
    x.l0 = (local / ntok) * S::TL;
    // The group's rows are divided evenly among its tiles: a last tile of a few
    // rows would load as many weights as a full one.
    const int rows = start[x.g + 1] - start[x.g];
    const int each = ((rows - 1) / ntok + S::NMMA_STEP) & ~(S::NMMA_STEP - 1);
    const int first = (local % ntok) * each;
    x.r0 = start[x.g] + first;
    x.n0 = first;
    x.nv = min(each, rows - first);
    x.klen = a.k;
  }
  if (a.out.alpha == 0.0f) x.klen = 0;
  x.any = x.klen > 0;
  x.end = 0;
  if (MODE == INNER) {
    if (rank % S::P == S::P - 1 || S::P == 1) x.end = x.klen & 15;
    x.klen &= ~15;
  }
  x.kt = (x.klen + BK - 1) / BK;
  x.k_lo = S::P > 1 ? (int)((int64_t)x.kt * rank / S::P) : 0;
  x.k_hi = S::P > 1 ? (int)((int64_t)x.kt * (rank + 1) / S::P) : x.kt;
  return x;
}

// The lines past a group's last row hold the next group's (whatever they are,
// infinities among them): zeroes lines `left` .. 15 of `chunks` 64-element chunks
// of 16 lines. A whole warp calls it.
__device__ __forceinline__ void zero_end(uint8_t *st, int left, int chunks, int lane) {
  for (int q = 0; q < chunks; q++)
    for (int r = left + (lane >> 3); r < 16; r += 4)
      *reinterpret_cast<uint4 *>(st + q * 2048 + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
  wgtc::fence_proxy_async_smem();
  __syncwarp();
}

// DRAIN: k-blocks after which an accumulator is drained (SEG, LONG; 0: at the tile's end).
// Warps: 0 and 10 load (the L and the N side), 1 issues the MMAs, 2-9 store, 11
// (inner form) zeroes what is past a group's last row. That a group ends inside
// the 16 lines of an MMA is known when its tile begins: those lines go to a place
// of their own, loaded ahead of the tile's k-blocks and multiplied after them, so
// that landing, zeroing and (in a pair) telling the other CTA are out of the way.
// (With the last block zeroed in the ring they cost 27 us of 145 at 8192 rows in
// 8 groups, 2048 x 4096 results.)
template <int MODE, class S, int DRAIN>
__global__ void __launch_bounds__(MODE == INNER ? 384 : 352, 1)
grouped_kernel(const __grid_constant__ CUtensorMap map_l, const __grid_constant__ CUtensorMap map_n,
               const __grid_constant__ CUtensorMap map_el, const __grid_constant__ CUtensorMap map_en, const Args a) {
  constexpr bool L_MN = MODE != ROWS_T, N_MN = MODE == INNER;
  constexpr int STAGES = S::STAGES, CG = S::CG;
  constexpr int NBOX = S::BN < 64 ? S::BN : 64;  // lines of one N-side box
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = wgtc::smem_addr(smem_raw);
  uint8_t *smem = smem_raw + ((1024 - (base & 1023)) & 1023);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + S::bars);
  uint64_t *empty = full + STAGES;
  constexpr int ENDS = S::ENDS;
  uint64_t *end_here = empty + STAGES;   // [ENDS] a group's last lines have landed in this CTA
  uint64_t *end_peer = end_here + ENDS;  // ... the other CTA of a pair has zeroed what is past them
  uint64_t *end_full = end_peer + ENDS;  // ... both have
  uint64_t *end_empty = end_full + ENDS;
  uint64_t *acc_full = end_empty + ENDS;    // [2]
  uint64_t *acc_empty = acc_full + 2;       // [2]
  wgg::Parts parts = {reinterpret_cast<float *>(smem + S::parts), acc_empty + 2, acc_empty + 3, 0};
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 4);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  int *start = reinterpret_cast<int *>(smem + S::tables);
  int *tile0 = start + a.groups + 1;

  const int warp = wgg::warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = S::CLUSTER > 1 ? wgtc::cluster_ctarank() : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      wgtc::mbar_init(&full[s], 2);
      wgtc::mbar_init(&empty[s], 1);
    }
    for (int e = 0; e < ENDS; e++) {
      wgtc::mbar_init(&end_here[e], 2);
      wgtc::mbar_init(&end_peer[e], 1);
      wgtc::mbar_init(&end_full[e], 1);
      wgtc::mbar_init(&end_empty[e], 1);
    }
    for (int b = 0; b < 2; b++) {
      wgtc::mbar_init(&acc_full[b], 1);
      wgtc::mbar_init(&acc_empty[b], CG * EPI_WARPS);
    }
    wgtc::mbar_init(parts.full, 1);
    wgtc::mbar_init(parts.empty, EPI_WARPS);
    *abort_flag = 0;
    wgtc::fence_barrier_init();
  }
  if (warp == 0 && lane == 0) wgtc::prefetch_tensormap(&map_l);
  if (warp == 10 && lane == 0) wgtc::prefetch_tensormap(&map_n);
  if (warp == 1) wgg::pair_tmem_alloc<CG>(tmem_slot, 2 * S::BN);
  wg_pdl_wait();
  wg_pdl_trigger();
  wgg::plan_groups(a.offsets, a.groups, a.rows, S::BN, start, MODE == INNER ? nullptr : tile0, nullptr, a.dwords);
  wgtc::tc_fence_before();
  wgg::cluster_sync<S::CLUSTER>();
  wgtc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int64_t tiles = MODE == INNER ? (int64_t)a.groups * a.tiles_l * a.tiles_n
                                      : (int64_t)tile0[a.groups] * a.tiles_l;
  const int64_t t_first = blockIdx.x / S::CLUSTER, t_step = gridDim.x / S::CLUSTER;
  const uint32_t half = CG == 2 ? rank : 0;  // which lanes and columns of a pair's tile

  // A wait that gives up records it and tells the other roles to stop at their
  // next failed wait (each is bounded on its own).
  auto gave_up = [&](unsigned bit) {
    atomicOr(a.dwords + WG_DW_ERROR, bit);
    *abort_flag = 1;
  };

  if (warp == 0 || warp == 10) {
    // ---- producers: each CTA of a pair loads its own lanes and its half of the columns ----
    wgg::Ring<STAGES> ring;
    wgg::Ring<ENDS> ends;
    bool ok = true;
    const bool l_side = warp == 0;
    const uint32_t lead = wgg::leader_addr<CG>(full);
    for (int64_t t = t_first; t < tiles && ok; t += t_step) {
      const Tile x = tile_at<MODE, S>(a, t, start, tile0, rank);
      const int cols = ((x.nv + S::NMMA_STEP - 1) & ~(S::NMMA_STEP - 1)) / CG;  // columns this CTA loads
      // The first box's outer coordinate, and how many boxes.
      const int c0 = l_side ? x.l0 + (int)half * BL : (N_MN ? x.n0 : x.r0) + (int)half * cols;
      const int boxes = l_side ? 2 : (cols + NBOX - 1) / NBOX;
      const uint32_t bytes = (uint32_t)(l_side ? S::L_BYTES : boxes * NBOX * 128);
      const int lg = x.g * a.l_group;
      if (MODE == INNER && x.end) {
        const int e = ends.s;
        ok = __all_sync(0xffffffffu, wgtc::mbar_wait_bounded(&end_empty[e], ends.round ^ 1u, WAIT_BUDGET));
        if (!ok) break;
        if (wgg::elect()) {
          uint8_t *dst = smem + S::ends + (size_t)e * S::END + (l_side ? 0 : 2 * 2048);
          wgtc::mbar_arrive_expect_tx(&end_here[e], (uint32_t)boxes * 2048);
          for (int b = 0; b < boxes; b++)
            wgtc::tma_load_2d(dst + b * 2048, l_side ? &map_el : &map_en, &end_here[e], c0 + b * 64, x.r0 + x.klen);
        }
        __syncwarp();
        ends.next();
      }
      for (int kb = x.k_lo; kb < x.k_hi; kb++, ring.next()) {
        const int s = ring.s;
        ok = wgtc::mbar_wait_bounded(&empty[s], ring.round ^ 1u, WAIT_BUDGET);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        uint8_t *dst = smem + (size_t)s * S::STAGE + (l_side ? 0 : S::L_BYTES);
        const int k0 = (MODE == INNER ? x.r0 : 0) + kb * BK;
        const uint32_t at = lead + 8u * (uint32_t)s;
        if (wgg::elect()) {
          if (half == 0) wgtc::mbar_arrive_expect_tx(&full[s], CG * bytes);
          if (l_side) {
            if (MODE == ROWS_T) {
              wgg::load_3d<CG>(dst, &map_l, &full[s], at, k0, c0, lg);
            } else if (MODE == ROWS_N) {
              wgg::load_3d<CG>(dst, &map_l, &full[s], at, c0, k0, lg);
              wgg::load_3d<CG>(dst + CHUNK, &map_l, &full[s], at, c0 + 64, k0, lg);
            } else {
              wgg::load_2d<CG>(dst, &map_l, &full[s], at, c0, k0);
              wgg::load_2d<CG>(dst + CHUNK, &map_l, &full[s], at, c0 + 64, k0);
            }
          } else {
            for (int b = 0; b < boxes; b++) {
              if (N_MN) wgg::load_2d<CG>(dst + b * CHUNK, &map_n, &full[s], at, c0 + b * 64, k0);
              else wgg::load_2d<CG>(dst + b * NBOX * 128, &map_n, &full[s], at, k0, c0 + b * NBOX);
            }
          }
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) gave_up(WG_DERR_TMA_WAIT);
    // Let every copy (of both CTAs) land before the CTA can exit: the MMAs that
    // read a stage complete after its copies, and free it.
    for (int i = 0; i < STAGES && ok; i++, ring.next())
      if (!wgtc::mbar_wait_bounded(&empty[ring.s], ring.round ^ 1u, WAIT_BUDGET)) break;
    for (int i = 0; i < ENDS && ok; i++, ends.next())
      if (!wgtc::mbar_wait_bounded(&end_empty[ends.s], ends.round ^ 1u, WAIT_BUDGET)) break;
  } else if (MODE == INNER && warp == 11) {
    // ---- ragged ends: zeroes the lines past a group's last row, then hands the place on ----
    // Lines are loaded behind the k-blocks of the tiles before theirs, so a wait lasts as long
    // as those take: 2^24 k-blocks pass the limit that the other waits have. This one's
    // grows with them, by ten times what a k-block takes.
    wgg::Ring<ENDS> ends;
    long long budget = WAIT_BUDGET;
    for (int64_t t = t_first; t < tiles; t += t_step) {
      const Tile x = tile_at<MODE, S>(a, t, start, tile0, rank);
      const long long blocks = x.k_hi - x.k_lo;
      if (!x.end) {
        budget += blocks * BLOCK_BUDGET;
        continue;
      }
      const int e = ends.s;
      const int nmma = (x.nv + S::NMMA_STEP - 1) & ~(S::NMMA_STEP - 1);
      bool ok = __all_sync(0xffffffffu, wgtc::mbar_wait_bounded(&end_here[e], ends.round, budget));
      budget = WAIT_BUDGET + blocks * BLOCK_BUDGET;
      if (ok) {
        zero_end(smem + S::ends + (size_t)e * S::END, x.end, 2 + (nmma / CG + 63) / 64, lane);
        if (CG == 2 && half == 1) {
          if (lane == 0) wgtc::mbar_arrive_cluster(wgtc::mapa_shared(wgtc::smem_addr(&end_peer[e]), 0));
        } else {
          if (CG == 2)
            ok = __all_sync(0xffffffffu, wgtc::mbar_wait_bounded_cluster(&end_peer[e], ends.round, WAIT_BUDGET));
          if (ok && lane == 0) mbar_arrive(&end_full[e]);
        }
      }
      if (!ok) {
        if (lane == 0) gave_up(WG_DERR_TMA_WAIT);
        break;
      }
      ends.next();
    }
  } else if (warp == 1) {
    if (half == 0) {
      // ---- MMA issuer ----
      wgg::Ring<STAGES> ring;
      wgg::Ring<ENDS> ends;
      int used = 0;
      constexpr int segment = DRAIN ? DRAIN : 1 << 30;
      constexpr uint64_t step_l = (L_MN ? 2048 : 32) >> 4, step_n = (N_MN ? 2048 : 32) >> 4;
      const uint32_t smem0 = wgtc::smem_addr(smem);
      const uint64_t desc_l0 = L_MN ? smem_desc_mn(smem0) : wgtc::smem_desc_kmajor(smem0, 128);
      const uint64_t desc_n0 = N_MN ? smem_desc_mn(smem0 + S::L_BYTES) : wgtc::smem_desc_kmajor(smem0 + S::L_BYTES, 128);
      bool ok = true;
      for (int64_t t = t_first; t < tiles && ok; t += t_step) {
        const Tile x = tile_at<MODE, S>(a, t, start, tile0, rank);
        const int nmma = (x.nv + S::NMMA_STEP - 1) & ~(S::NMMA_STEP - 1);
        const uint32_t idesc = idesc_f16(a.ab_format, S::TL, nmma, L_MN, N_MN);
        if (x.k_hi == x.k_lo && !x.end) continue;
        int kb0 = x.k_lo;
        do {  // a segment (one without k-blocks when there is nothing but an end)
          const int b = used & 1, kb1 = min(x.k_hi, kb0 + segment);
          const bool end = x.end && kb1 == x.k_hi;
          const uint32_t d_tmem = tmem + (uint32_t)(b * S::BN);
          ok = __all_sync(0xffffffffu, wgg::leader_wait<CG>(&acc_empty[b], ((uint32_t)(used >> 1) & 1u) ^ 1u));
          wgtc::tc_fence_after();
          for (int kb = kb0; kb < kb1 && ok; kb++, ring.next()) {
            ok = __all_sync(0xffffffffu, wgtc::mbar_wait_bounded(&full[ring.s], ring.round, WAIT_BUDGET));
            if (!ok) break;
            wgtc::tc_fence_after();
            const uint64_t at = (uint64_t)((uint32_t)ring.s * (S::STAGE >> 4));
            const uint64_t dl = desc_l0 + at, dn = desc_n0 + at;
            const int steps = (x.klen - kb * BK + 15) >> 4;
            if (wgg::elect()) {
              if (steps >= 4) {
#pragma unroll
                for (int kk = 0; kk < 4; kk++)
                  mma_f16<CG>(d_tmem, dl + kk * step_l, dn + kk * step_n, idesc, kk > 0 || kb > kb0 ? 1u : 0u);
              } else {
                for (int kk = 0; kk < steps; kk++)
                  mma_f16<CG>(d_tmem, dl + kk * step_l, dn + kk * step_n, idesc, kk > 0 || kb > kb0 ? 1u : 0u);
              }
              wgg::commit<CG>(&empty[ring.s]);
              if (kb == kb1 - 1 && !end) wgg::commit<CG>(&acc_full[b]);
            }
            __syncwarp();
          }
          if (MODE == INNER && ok && end) {
            ok = __all_sync(0xffffffffu, wgtc::mbar_wait_bounded(&end_full[ends.s], ends.round, WAIT_BUDGET));
            if (!ok) break;
            wgtc::tc_fence_after();
            const uint32_t at = smem0 + (uint32_t)S::ends + (uint32_t)(ends.s * S::END);
            if (wgg::elect()) {
              mma_f16<CG>(d_tmem, smem_desc_mn(at, 2048), smem_desc_mn(at + 2 * 2048, 2048), idesc, kb1 > kb0 ? 1u : 0u);
              wgg::commit<CG>(&end_empty[ends.s]);
              wgg::commit<CG>(&acc_full[b]);
            }
            __syncwarp();
            ends.next();
          }
          kb0 += segment;
          used++;
        } while (kb0 < x.k_hi && ok);
      }
      if (!ok && lane == 0) gave_up(WG_DERR_MMA_WAIT);
    }
  } else if (warp >= 2 && warp < 2 + EPI_WARPS) {
    // ---- epilogue ----
    const int q = warp & 3, h = (warp - 2) >> 2;
    int used = 0;
    bool ok = true;
    auto wait_acc = [&](int b) {
      bool got = wgtc::mbar_wait_bounded(&acc_full[b], (uint32_t)(used >> 1) & 1u, WAIT_BUDGET) && *abort_flag == 0;
      got = __all_sync(0xffffffffu, got);
      if (!got && lane == 0) gave_up(WG_DERR_MMA_WAIT);
      wgtc::tc_fence_after();
      return got;
    };
    auto free_acc = [&](int b) {
      wgtc::tc_fence_before();
      __syncwarp();
      if (lane == 0) wgg::leader_arrive<CG>(&acc_empty[b]);
      used++;
    };
    for (int64_t t = t_first; t < tiles && ok; t += t_step) {
      const Tile x = tile_at<MODE, S>(a, t, start, tile0, rank);
      const int valid = x.nv - h * S::CPT;  // columns this warp has (may be none)
      const int l = x.l0 + (int)half * BL + q * 32 + lane;
      const int64_t row = (MODE == INNER ? x.n0 : x.r0) + h * S::CPT;
      const int64_t at = (MODE == INNER ? (int64_t)x.g * a.strideC : 0) + row * a.out.ldc + l;
      const uint32_t col = tmem + (uint32_t)(h * S::CPT) + ((uint32_t)(q * 32) << 16);
      if constexpr (DRAIN) {
        float sum[S::CPT];
#pragma unroll
        for (int j = 0; j < S::CPT; j++) sum[j] = 0.0f;
        for (int kb0 = x.k_lo; kb0 < x.k_hi || (kb0 == x.k_lo && x.end); kb0 += DRAIN) {
          const int b = used & 1;
          if (!(ok = wait_acc(b))) break;
          wgg::drain<S::CPT>(col + (uint32_t)(b * S::BN), valid, kb0 == x.k_lo, sum);
          free_acc(b);
        }
        if (!ok) break;
        bool mine = true;
        if constexpr (S::P > 1) {
          if (x.any) mine = wgg::join_parts<S::P, S::BN, S::CPT>(parts, rank, h * S::CPT, q * 32 + lane, valid, x.nv,
                                                                         warp == 2, t + t_step < tiles, sum, &ok);
          else mine = rank == 0;
          if (!ok) {
            if (lane == 0) gave_up(WG_DERR_MMA_WAIT);
            break;
          }
        }
        if (mine) wgg::store_sums<S::CPT, DRAIN == SEG && S::P == 1>(a.out, at, l < a.nl, valid, sum);
      } else {
        const int b = used & 1;
        if (x.any && !(ok = wait_acc(b))) break;
        wgg::store_acc<S::CPT>(col + (uint32_t)(b * S::BN), x.any, a.out, at, l < a.nl, valid);
        if (x.any) free_acc(b);
      }
    }
  }

  wgtc::tc_fence_before();
  __syncwarp();
  wgg::cluster_sync<S::CLUSTER>();
  if (warp == 1) {
    wgtc::tc_fence_after();
    wgg::pair_tmem_dealloc<CG>(tmem, 2 * S::BN);
  }
}

// ---- rows of any alignment to rows of whole 16-byte units --------------------

struct Realign {
  const uint16_t *src, *end;  // the matrices' first element, and behind their last
  uint16_t *dst;
  int64_t ld, stride, ld_out;
  int64_t lines;      // rows of all matrices together
  int rows, cols;     // of one matrix
  const int *offsets;  // matrices of groups without rows are not copied (NULL: all are)
};

// Eight elements that begin s elements into the 16-byte unit a; b is the next unit.
__device__ __forceinline__ uint4 shifted(const uint4 &a, const uint4 &b, int s) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (s & 2)
#pragma unroll
    for (int i = 0; i < 7; i++) w[i] = w[i + 1];
  if (s & 4)
#pragma unroll
    for (int i = 0; i < 6; i++) w[i] = w[i + 2];
  const int sh = (s & 1) * 16;
  return make_uint4(__funnelshift_r(w[0], w[1], sh), __funnelshift_r(w[1], w[2], sh),
                    __funnelshift_r(w[2], w[3], sh), __funnelshift_r(w[3], w[4], sh));
}

// A warp a line: aligned 16-byte loads, moved into place by words and half words.
// Bound by latency, so a thread's four pairs of loads go out together (20 MB cold: 10.4
// us; one pair after the other 15.8). Memory outside the matrices is not read. What
// follows a line's last element in its last unit is never read (the tensor maps end at
// `cols`).
__global__ void __launch_bounds__(256) grouped_realign(const Realign x, const Realign y) {
  constexpr int U = 4;
  wg_pdl_wait();
  wg_pdl_trigger();
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const bool second = w >= x.lines;
  const Realign &a = second ? y : x;
  const int64_t line = second ? w - x.lines : w;
  if (line >= a.lines) return;
  const int64_t g = line >> 32 ? line / a.rows : (uint32_t)line / (uint32_t)a.rows, r = line - g * a.rows;
  if (a.offsets && a.offsets[g + 1] <= a.offsets[g]) return;
  const uint16_t *src = a.src + g * a.stride + r * a.ld;
  const int s = (int)(reinterpret_cast<uintptr_t>(src) & 15) >> 1;  // the line's place in its first unit
  const uint16_t *base = src - s, *lo = a.src, *hi = a.end;
  uint16_t *dst = a.dst + line * a.ld_out;
  for (int e = (threadIdx.x & 31) * 8; e < a.cols; e += 256 * U) {
    uint4 p[U], q[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const uint16_t *at = base + e + 256 * u;
      const bool use = e + 256 * u < a.cols;
      p[u] = q[u] = make_uint4(0, 0, 0, 0);
      if (use && at >= lo && at + 8 <= hi) p[u] = __ldg(reinterpret_cast<const uint4 *>(at));
      if (use && s && at + 16 <= hi) q[u] = __ldg(reinterpret_cast<const uint4 *>(at + 8));
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = e + 256 * u;
      if (c >= a.cols) continue;
      const uint16_t *at = base + c;
      uint4 v = shifted(p[u], q[u], s);
      if (at < lo || at + (s ? 16 : 8) > hi) {  // at an end of the matrices: element by element
        uint32_t h[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (c + i < a.cols) h[i >> 1] |= (uint32_t)__ldg(src + c + i) << (16 * (i & 1));
        v = make_uint4(h[0], h[1], h[2], h[3]);
      }
      *reinterpret_cast<uint4 *>(dst + c) = v;
    }
  }
}

constexpr int64_t LIM = (int64_t)1 << 31;

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

// A TMA map can read row-major matrices whose base, row length and distance are
// whole 16-byte units (cuTensorMapEncodeTiled's rule; strides below 2^40 bytes).
bool mappable(const void *p, int64_t ld, int64_t stride) {
  return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && stride % 8 == 0 && ld < ((int64_t)1 << 39) &&
         stride < ((int64_t)1 << 39);
}

// The tensor maps of a call (mappable operands).
template <int MODE, class S>
bool make_maps(const Args &a, int type, CUtensorMap *ml, CUtensorMap *mn, CUtensorMap *el, CUtensorMap *en) {
  const cuuint64_t ldl = (cuuint64_t)a.ldl * 2, ldn = (cuuint64_t)a.ldn * 2;
  if (MODE == INNER) {
    const cuuint64_t dl[2] = {(cuuint64_t)a.nl, (cuuint64_t)a.rows}, dn[2] = {(cuuint64_t)a.nn, (cuuint64_t)a.rows};
    const cuuint32_t box[2] = {64, 64};
    const cuuint32_t end[2] = {64, 16};
    return encode(ml, type, a.L, 2, dl, &ldl, box) && encode(mn, type, a.N, 2, dn, &ldn, box) &&
           encode(el, type, a.L, 2, dl, &ldl, end) && encode(en, type, a.N, 2, dn, &ldn, end);
  }
  const int64_t lrows = MODE == ROWS_T ? a.nl : a.k, lcols = MODE == ROWS_T ? a.k : a.nl;
  const cuuint64_t dl[3] = {(cuuint64_t)lcols, (cuuint64_t)lrows, a.l_group ? (cuuint64_t)a.groups : 1};
  const cuuint64_t sl[2] = {ldl, a.l_group ? (cuuint64_t)a.strideL * 2 : ldl * (cuuint64_t)lrows};
  const cuuint32_t bl[3] = {64, MODE == ROWS_T ? (cuuint32_t)BL : 64u, 1};
  const cuuint64_t dn[2] = {(cuuint64_t)a.k, (cuuint64_t)a.rows};
  const cuuint32_t bn[2] = {64, (cuuint32_t)std::min(S::BN, 64)};
  return encode(ml, type, a.L, 3, dl, sl, bl) && encode(mn, type, a.N, 2, dn, &ldn, bn);
}

template <int MODE, class S, int DRAIN>
wg_status launch_as(wg_device *d, Args &a, const CUtensorMap (&m)[4]) {
  a.tiles_l = (a.nl + S::TL - 1) / S::TL;
  a.tiles_n = MODE == INNER ? (a.nn + S::BN - 1) / S::BN : 0;
  const int64_t most = (int64_t)a.tiles_l * (MODE == INNER ? (int64_t)a.groups * a.tiles_n
                                                           : (int64_t)a.rows / S::BN + a.groups);
  const unsigned grid = S::CLUSTER * (unsigned)std::max<int64_t>(1, std::min<int64_t>(most, d->sm_count / S::CLUSTER));
  wg_launch_scope scope(d, MODE == INNER ? "gemm_grouped_inner" : "gemm_grouped");
  WG_CUDA(wg_kernel_smem(grouped_kernel<MODE, S, DRAIN>, SMEM_LIMIT));
  WG_CUDA((wgg::launch<S::CLUSTER>(grouped_kernel<MODE, S, DRAIN>, grid, MODE == INNER ? 384 : 352, S::smem(a.groups),
                              d->stream, m[0], m[1], m[2], m[3], a)));
  WG_CUDA(cudaGetLastError());
  return WG_OK;
}

template <int MODE, class S>
wg_status launch(wg_device *d, Args &a, int type) {
  CUtensorMap m[4];
  memset(m, 0, sizeof m);
  // (no product, no operands)
  if (a.out.alpha != 0.0f && !make_maps<MODE, S>(a, type, &m[0], &m[1], &m[2], &m[3]))
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "the operands' sizes exceed what a tensor map describes");
  // (a split contraction's sums are always drained, and few blocks long)
  if constexpr (S::P > 1) {
    return launch_as<MODE, S, SEG>(d, a, m);
  } else {
    const int rows = MODE == INNER ? a.rows : a.k;  // the longest contraction there can be
    if (a.out.type == WG_TYPE_F32) return rows > SEG * BK ? launch_as<MODE, S, SEG>(d, a, m) : launch_as<MODE, S, 0>(d, a, m);
    return rows > whole_rows(a.out.type) ? launch_as<MODE, S, LONG>(d, a, m) : launch_as<MODE, S, 0>(d, a, m);
  }
}

// The form with the least modelled time. A form's tiles run in rounds over the
// SMs; a round takes its k-blocks times the larger of the tensor core's time and
// the time an SM needs to receive the block (65 bytes a clock from L2), or the
// clocks that issuing it takes; joining a split contraction adds a fixed time.
// Groups are taken to be evenly filled: the host does not know their sizes. us in
// a CUDA graph, operands in L2, m x n x k (groups), the chosen form's starred:
//                           pair   128 columns   64      32     64/2    32/2    32/4
//   4 x 512 x 4096 (8)      16.0      15.9      15.6    15.6    10.8    10.7     7.8*
//   64 x 4096 x 4096 (1)    16.6      16.6      16.3    15.9    12.8    11.6*   17.4
//   8 x 1024 x 2048 (8)     10.2      10.3      10.1     9.6    10.6     8.9*   13.5
//   512 x 512 x 512 (1)      7.8       5.7       5.0     4.9*    6.7     5.8    11.8
//   1024 x 1024 x 1024 (1)  10.3       7.7       7.0*   10.2    10.2    12.6    28.1
//   1000 x 1024 x 776 (7)   10.4       9.0*     11.2    10.4    12.6    13.2    29.4
//   2000 x 2048 x 2048 (8)  16.6*     20.8      32.7    51.2    34.9    58.5   129
enum Form { PAIR_256, ONE_128, ONE_64, ONE_32, SPLIT_64, SPLIT_32_2, SPLIT_32_4, FORMS };
template <int MODE>
Form choose(const wg_device *d, const Args &a) {
  static const struct { int cg, bn, p; } forms[FORMS] = {{2, 256, 1}, {1, 128, 1}, {1, 64, 1}, {1, 32, 1},
                                                         {1, 64, 2}, {1, 32, 2}, {1, 32, 4}};
  const int64_t groups = MODE == INNER ? a.groups : std::max<int64_t>(1, std::min(a.groups, a.rows));
  const int64_t cols = MODE == INNER ? a.nn : (a.rows + groups - 1) / groups;  // of one group
  const int64_t klen = MODE == INNER ? (a.rows + groups - 1) / groups : a.k;
  const int64_t kt = std::max<int64_t>(1, (klen + BK - 1) / BK);
  Form best = ONE_128;
  double least = 1e300;
  for (int i = 0; i < FORMS; i++) {
    const auto f = forms[i];
    if (MODE == INNER && f.bn < 64) continue;
    const int64_t nt = (cols + f.bn - 1) / f.bn, nv = MODE == INNER ? std::min<int64_t>(cols, f.bn) : (cols + nt - 1) / nt;
    const int64_t tl = (a.nl + f.cg * BL - 1) / (f.cg * BL), slots = f.p == 4 ? d->sm_count * 7 / 32 : d->sm_count / (f.cg * f.p);
    const int64_t rounds = (tl * groups * nt + slots - 1) / slots;
    const int64_t box = std::min<int64_t>(f.bn, 64), lines = (nv / f.cg + box - 1) / box * box;
    const double mma = nv * 2.0;  // 4 MMAs of 16: 2 clocks a column (128 or 256 lanes)
    const double block = std::max({mma, (BL + lines) * 128 / 65.0, 230.0});
    // A tile's results: the last round's are stored in the open (20 bytes a clock).
    const double tail = (double)BL * nv * (a.out.type == WG_TYPE_F32 ? 4 : 2) / 20 + (f.p > 1 ? 1800 : 0);
    const double t = rounds * (double)((kt + f.p - 1) / f.p) * block + tail;
    if (t < least) {
      least = t;
      best = (Form)i;
    }
  }
  return best;
}

template <int MODE>
wg_status run(wg_device *d, Args &a, int type) {
  // Weights shared by all groups (stride 0, or one group) need no group dimension.
  a.l_group = MODE != INNER && a.groups > 1 && a.strideL != 0;
  wg_temp temp;
  if (a.out.alpha != 0.0f) {
    Realign l = {}, n = {};
    size_t bytes = 0;
    if (!mappable(a.L, a.ldl, a.l_group ? a.strideL : 0)) {
      l.src = a.L;
      l.ld = a.ldl;
      l.stride = a.l_group ? a.strideL : 0;
      l.rows = MODE == INNER ? a.rows : MODE == ROWS_T ? a.nl : a.k;
      l.cols = MODE == ROWS_T ? a.k : a.nl;
      l.lines = (int64_t)l.rows * (a.l_group ? a.groups : 1);
      l.ld_out = ((int64_t)l.cols + 7) / 8 * 8;
      l.end = l.src + (l.lines / l.rows - 1) * l.stride + (int64_t)(l.rows - 1) * l.ld + l.cols;
      l.offsets = a.l_group ? a.offsets : nullptr;
      bytes = (size_t)(l.lines * l.ld_out) * 2;
    }
    if (!mappable(a.N, a.ldn, 0)) {
      n.src = a.N;
      n.ld = a.ldn;
      n.rows = a.rows;
      n.cols = MODE == INNER ? a.nn : a.k;
      n.lines = n.rows;
      n.ld_out = ((int64_t)n.cols + 7) / 8 * 8;
      n.end = n.src + (int64_t)(n.rows - 1) * n.ld + n.cols;
    }
    const size_t total = bytes + (size_t)(n.lines * n.ld_out) * 2;
    if (total) {
      wg_status st = wg_temp_get(d, total, &temp);
      if (st != WG_OK) return st;
      if (l.lines) {
        l.dst = static_cast<uint16_t *>(temp.ptr);
        a.L = l.dst;
        a.ldl = l.ld_out;
        if (a.l_group) a.strideL = l.rows * l.ld_out;
      }
      if (n.lines) {
        n.dst = reinterpret_cast<uint16_t *>(static_cast<char *>(temp.ptr) + bytes);
        a.N = n.dst;
        a.ldn = n.ld_out;
      }
      const int64_t blocks = (l.lines + n.lines + 7) / 8;
      cudaError_t e = blocks < LIM ? cudaSuccess : cudaErrorInvalidValue;
      if (e == cudaSuccess) {
        wg_launch_scope scope(d, "grouped_realign");
        e = wg_launch_pdl(grouped_realign, dim3((unsigned)blocks), dim3(256), 0, d->stream, l, n);
      }
      if (e != cudaSuccess) {
        wg_temp_done(d, &temp);
        return wg_fail(WG_ERR_CUDA, "grouped_realign failed: %s", cudaGetErrorString(e));
      }
    }
  }
  wg_status st;
  const Form form = choose<MODE>(d, a);
  switch (form) {
    case PAIR_256: st = launch<MODE, Shape<2, 256>>(d, a, type); break;
    case ONE_128: st = launch<MODE, Shape<1, 128>>(d, a, type); break;
    case ONE_64: st = launch<MODE, Shape<1, 64>>(d, a, type); break;
    case SPLIT_64: st = launch<MODE, Shape<1, 64, 2>>(d, a, type); break;
    default:
      if constexpr (MODE == INNER) {
        st = WG_ERR_INVALID_ARGUMENT;  // (not chosen: 64 columns are the least an MN-major side has)
      } else {
        st = form == ONE_32 ? launch<MODE, Shape<1, 32>>(d, a, type)
             : form == SPLIT_32_2 ? launch<MODE, Shape<1, 32, 2>>(d, a, type)
                               : launch<MODE, Shape<1, 32, 4>>(d, a, type);
      }
  }
  const wg_status done = wg_temp_done(d, &temp);
  return st == WG_OK ? done : st;
}

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

wg_status check_pointers(const void *A, const void *B, const void *C, int type, int ctype, const int *offsets) {
  wg_status st;
  if ((st = wgg::check_aligned("A", A, type)) != WG_OK || (st = wgg::check_aligned("B", B, type)) != WG_OK ||
      (st = wgg::check_aligned("C", C, ctype)) != WG_OK)
    return st;
  return wgg::check_offsets(offsets);
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
  if ((st = check_pointers(A, B, C, type, ctype, offsets)) != WG_OK) return st;
  st = wgg::check_arch(d);
  if (st != WG_OK) return st;
  if (beta == 1.0f && (alpha == 0.0f || k == 0)) return WG_OK;  // C stays as it is
  wg_device_guard guard(d->ordinal);
  Args a = {};
  a.groups = (int)groups;
  a.rows = (int)m;
  a.nl = (int)n;
  a.k = (int)k;
  a.offsets = offsets;
  a.out = {C, ldc, k > 0 ? alpha : 0.0f, beta, ctype};
  a.ab_format = type == WG_TYPE_BF16 ? 1u : 0u;
  a.L = static_cast<const uint16_t *>(B);
  a.ldl = ldb;
  a.strideL = strideB;
  a.N = static_cast<const uint16_t *>(A);
  a.ldn = lda;
  a.dwords = d->dwords;
  return wg_timed(d, gpu_ms, [&] { return transB ? run<ROWS_T>(d, a, type) : run<ROWS_N>(d, a, type); });
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
  if (groups > 1 && (strideC < 0 || !wgg::apart(strideC, m, n, ldc) || strideC >= ((int64_t)1 << 40)))
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "strideC must be at least one matrix of C and below 2^40.");
  if (groups == 0 || m == 0 || n == 0) return WG_OK;
  if (!offsets || !C || (k > 0 && alpha != 0.0f && (!A || !B)))
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "operand pointer is NULL");
  if ((st = check_pointers(A, B, C, type, ctype, offsets)) != WG_OK) return st;
  st = wgg::check_arch(d);
  if (st != WG_OK) return st;
  if (beta == 1.0f && (alpha == 0.0f || k == 0)) return WG_OK;  // C stays as it is
  wg_device_guard guard(d->ordinal);
  Args a = {};
  a.groups = (int)groups;
  a.rows = (int)k;
  a.nl = (int)n;
  a.nn = (int)m;
  a.offsets = offsets;
  a.strideC = groups > 1 ? strideC : 0;
  a.out = {C, ldc, k > 0 ? alpha : 0.0f, beta, ctype};
  a.ab_format = type == WG_TYPE_BF16 ? 1u : 0u;
  a.L = static_cast<const uint16_t *>(B);
  a.ldl = ldb;
  a.N = static_cast<const uint16_t *>(A);
  a.ldn = lda;
  a.dwords = d->dwords;
  return wg_timed(d, gpu_ms, [&] { return run<INNER>(d, a, type); });
}
