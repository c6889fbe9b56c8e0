// Microscaled 4-bit floating point (OCP MXFP4): quantisation, its inverse, and
// products on the tensor cores (tcgen05 kind::mxf4). wg_mx_* of the C ABI; no
// counterpart in the reference.
//
// Format. 32 neighbouring elements of a row share a scale 2^e held as the byte
// e + 127 (255: not a number); an element is sign, 2 exponent bits, 1 mantissa
// bit (0, .5, 1, 1.5, 2, 3, 4, 6). Quantising: e = floor(log2 max|x|) - 2 (the
// largest element, 6 = 1.5 * 2^2, has exponent 2), at least -127; x / 2^e is
// rounded to nearest, ties to even, what exceeds 6 to 6. A block with a NaN or an
// infinity gets the scale 255: everything computed from it is NaN.
//
// Storage. Codes two to a byte (the even column in the low half), each row
// padded to whole blocks (16 bytes each), padding zero. Scales in tiles of 128
// rows x 4 blocks, 512 bytes, so that one tile is what tcgen05.cp puts into TMEM
// for the MMA: row r, block b of a tile at byte 16 * (r % 32) + 4 * (r / 32) + b;
// tiles of one tile row follow one another along the columns; padding zero. In a
// matrix whose rows are grouped, every group's scales begin at a new tile row.
#include <algorithm>
#include <cstring>

#include "grouped_common.cuh"

namespace {

using wgg::BL;
using wgg::mbar_arrive;
using wgg::WAIT_BUDGET;

// ---- quantisation -----------------------------------------------------------

struct QuantArgs {
  const void *X;
  int64_t ldx, strideX;
  int xtype;
  int rows, cols;      // of the quantised matrix
  uint8_t *codes, *scales;
  int64_t pitch;       // bytes of a row of codes
  int tiles_r, tiles_c;  // scale tiles of one matrix
  int batch;
  const int *offsets;  // grouped rows (batch 1), or NULL
  int groups;
  unsigned *dwords;
};

// The scale byte of a block whose largest magnitude has these float32 bits.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255 ? 255u : (e > 2 ? e - 2 : 0u);
}
// 2^-e for the scale byte e + 127 (a normal float32 for every byte scale_byte gives).
__device__ __forceinline__ float inverse_scale(uint32_t byte) {
  return __uint_as_float((byte == 255 ? 127u : 254u - byte) << 23);
}
// 2^e; NaN for 255.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fffffffu : byte << 23);
}

// Eight float32 -> eight codes, element 0 in the lowest four bits.
__device__ __forceinline__ uint32_t encode8(const float (&x)[8]) {
  uint32_t out;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(out)
      : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
  return out;
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

// Eight elements at p of which the first `valid` exist, as float32.
template <class T>
__device__ __forceinline__ void load8(const T *p, int valid, float (&x)[8]) {
  if (valid >= 8 && ((uintptr_t)p & 15) == 0) {
    uint4 w[sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) w[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    const T *v = reinterpret_cast<const T *>(w);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = to_float(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = i < valid ? to_float(p[i]) : 0.0f;
  }
}

// The rows of one scale tile: first row, how many, and its matrix (batch).
struct TileRows {
  int r0, n, b;
};
// smem: start and atom0 tables of the groups (grouped matrices only).
__device__ __forceinline__ TileRows rows_of_tile(const QuantArgs &a, int tile, int *tables) {
  TileRows t;
  if (a.offsets) {
    int *start = tables, *atom0 = tables + a.groups + 1;
    wgg::plan_groups(a.offsets, a.groups, a.rows, 128, start, atom0, nullptr, a.dwords);
    t.b = 0;
    if (tile >= atom0[a.groups]) {
      t.r0 = t.n = 0;
      return t;
    }
    const int g = wgg::group_of(atom0, a.groups, tile);
    t.r0 = start[g] + (tile - atom0[g]) * 128;
    t.n = min(128, start[g + 1] - t.r0);
    return t;
  }
  t.b = tile / a.tiles_r;
  t.r0 = (tile - t.b * a.tiles_r) * 128;
  t.n = min(128, a.rows - t.r0);
  return t;
}

// One CTA per scale tile (128 rows x 128 columns): 16 threads a row, eight
// elements each, four threads a block; the tile's scales are gathered in shared
// memory and written as one piece.
template <class T>
__global__ void __launch_bounds__(256) mx_quantize(const QuantArgs a) {
  extern __shared__ int tables[];
  __shared__ __align__(16) uint8_t sf[512];
  wg_pdl_wait();
  wg_pdl_trigger();
  const int tile = (int)(blockIdx.x / (unsigned)a.tiles_c), tc = (int)(blockIdx.x % (unsigned)a.tiles_c);
  const TileRows t = rows_of_tile(a, tile, tables);
  if (t.n <= 0) return;
  if (threadIdx.x < 128) reinterpret_cast<uint32_t *>(sf)[threadIdx.x] = 0;
  __syncthreads();
  const T *X = static_cast<const T *>(a.X) + t.b * a.strideX;
  const int c = threadIdx.x & 15, col = tc * 128 + c * 8;
  const bool in = col / 32 * 16 < a.pitch;  // the block exists (it may end in padding)
  for (int r = threadIdx.x >> 4; r < t.n; r += 16) {
    const int64_t row = t.r0 + r;
    float x[8];
    load8(X + row * a.ldx + col, in ? a.cols - col : 0, x);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    // The loop's bound differs between rows: name the block's four lanes.
    const uint32_t four = 0xfu << (threadIdx.x & 28);
    top = max(top, __shfl_xor_sync(four, top, 1));
    top = max(top, __shfl_xor_sync(four, top, 2));
    const uint32_t e = scale_byte(top);
    const float inv = inverse_scale(e);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] *= inv;
    if (in) {
      const int64_t at = ((int64_t)t.b * a.rows + row) * a.pitch + col / 2;
      *reinterpret_cast<uint32_t *>(a.codes + at) = encode8(x);
      if ((c & 3) == 0) sf[(r & 31) * 16 + (r >> 5) * 4 + (c >> 2)] = (uint8_t)e;
    }
  }
  __syncthreads();
  if (threadIdx.x < 32)
    reinterpret_cast<uint4 *>(a.scales + ((int64_t)tile * a.tiles_c + tc) * 512)[threadIdx.x] =
        reinterpret_cast<const uint4 *>(sf)[threadIdx.x];
}

// The transposed form: X holds the matrix's columns as its rows. A thread takes
// one row of the result and 32 of X's rows; a warp's loads are 32 neighbouring
// elements.
template <class T>
__global__ void __launch_bounds__(256) mx_quantize_t(const QuantArgs a) {
  __shared__ __align__(16) uint8_t sf[512];
  wg_pdl_wait();
  wg_pdl_trigger();
  const int tile = (int)(blockIdx.x / (unsigned)a.tiles_c), tc = (int)(blockIdx.x % (unsigned)a.tiles_c);
  const TileRows t = rows_of_tile(a, tile, nullptr);
  if (threadIdx.x < 128) reinterpret_cast<uint32_t *>(sf)[threadIdx.x] = 0;
  __syncthreads();
  const T *X = static_cast<const T *>(a.X) + t.b * a.strideX;
  const int lane = threadIdx.x & 31;
  for (int w = threadIdx.x >> 5; w < 16; w += 8) {
    const int r = (w & 3) * 32 + lane, blk = w >> 2, col = tc * 128 + blk * 32;
    if (r >= t.n || col / 32 * 16 >= a.pitch) continue;
    float x[32];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) {
      x[i] = col + i < a.cols ? to_float(X[(int64_t)(col + i) * a.ldx + t.r0 + r]) : 0.0f;
      top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    }
    const uint32_t e = scale_byte(top);
    const float inv = inverse_scale(e);
    uint32_t code[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; j++) y[j] = x[i * 8 + j] * inv;
      code[i] = encode8(y);
    }
    const int64_t at = ((int64_t)t.b * a.rows + t.r0 + r) * a.pitch + col / 2;
    *reinterpret_cast<uint4 *>(a.codes + at) = make_uint4(code[0], code[1], code[2], code[3]);
    sf[(r & 31) * 16 + (r >> 5) * 4 + blk] = (uint8_t)e;
  }
  __syncthreads();
  if (threadIdx.x < 32)
    reinterpret_cast<uint4 *>(a.scales + ((int64_t)tile * a.tiles_c + tc) * 512)[threadIdx.x] =
        reinterpret_cast<const uint4 *>(sf)[threadIdx.x];
}

// ---- the values the codes stand for ------------------------------------------

// The value of a code times the scale (exact in float32: the magnitudes are
// multiples of a half below 8).
__device__ __forceinline__ float decode(uint32_t code, float scale) {
  const uint32_t m = code & 7u;
  // half steps: 0 1 2 3 4 6 8 12
  const float v = 0.5f * (float)(m < 5 ? m : m == 5 ? 6u : m == 6 ? 8u : 12u);
  return ((code & 8u) ? -v : v) * scale;
}

template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// X here is the output (rows x cols, ldx).
template <class T>
__global__ void __launch_bounds__(256) mx_dequantize(const QuantArgs a) {
  extern __shared__ int tables[];
  __shared__ __align__(16) uint8_t sf[512];
  wg_pdl_wait();
  wg_pdl_trigger();
  const int tile = (int)(blockIdx.x / (unsigned)a.tiles_c), tc = (int)(blockIdx.x % (unsigned)a.tiles_c);
  const TileRows t = rows_of_tile(a, tile, tables);
  if (t.n <= 0) return;
  if (threadIdx.x < 32)
    reinterpret_cast<uint4 *>(sf)[threadIdx.x] =
        reinterpret_cast<const uint4 *>(a.scales + ((int64_t)tile * a.tiles_c + tc) * 512)[threadIdx.x];
  __syncthreads();
  T *X = static_cast<T *>(const_cast<void *>(a.X)) + t.b * a.strideX;
  const int c = threadIdx.x & 15, col = tc * 128 + c * 8;
  if (col >= a.cols) return;
  for (int r = threadIdx.x >> 4; r < t.n; r += 16) {
    const int64_t row = t.r0 + r;
    const uint32_t code = *reinterpret_cast<const uint32_t *>(a.codes + ((int64_t)t.b * a.rows + row) * a.pitch + col / 2);
    const float s = scale_value(sf[(r & 31) * 16 + (r >> 5) * 4 + (c >> 2)]);
    T *p = X + row * a.ldx + col;
    alignas(16) T y[8];
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = from_float<T>(decode(code >> (4 * i) & 15u, s));
    if (col + 8 <= a.cols && ((uintptr_t)p & 15) == 0) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; i++)
        reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(y)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (col + i < a.cols) p[i] = y[i];
    }
  }
}

// ---- product ------------------------------------------------------------------
//
// The grouped kernel's frame and roles (grouped.cu): B's rows on the lanes, A's
// rows on the columns, both K-major. A k-block is 256 elements, 128 bytes of
// codes a row and two scale tiles of 128 rows for each operand; the MMA warp
// copies the scale tiles to TMEM (tcgen05.cp, four columns a tile) in front of
// the block's four MMAs of 64.

constexpr int BKE = 256;           // elements of a k-block
constexpr int EPI_WARPS = 4;
constexpr size_t SMEM_LIMIT = 227 * 1024;

template <int BN_>
struct Shape {
  static constexpr int BN = BN_;
  static constexpr int NT = BN / 128;            // scale tiles of the N side
  static constexpr int L_BYTES = BL * 128, N_BYTES = BN * 128;
  static constexpr int SF_L = 1024, SF_N = NT * 1024;
  static constexpr int STAGE = L_BYTES + N_BYTES + SF_L + SF_N;
  static constexpr int STAGES = (int)((SMEM_LIMIT - 12 * 1024) / STAGE);
  // TMEM columns: accumulators, then two sets of scales (L: 2 x 4, N: 2 x 4 NT).
  static constexpr int ACCS = BN <= 128 ? 2 : 1;
  static constexpr int SF_COL = ACCS * BN, SF_SET = 8 + 8 * NT;
  static constexpr int TMEM_COLS = 512;
  static_assert(SF_COL + 2 * SF_SET <= TMEM_COLS, "accumulators and scales must fit TMEM");
  static constexpr size_t smem(int groups) {
    return 1024 + (size_t)STAGES * STAGE + 256 + 3 * ((size_t)groups + 1) * sizeof(int);
  }
};

struct Args {
  int groups, rows, n, k;
  int tiles_l, katoms;
  int l_atoms;           // scale tile rows of one matrix of B
  const int *offsets;    // NULL: one group, all rows
  const uint8_t *sf_l, *sf_n;
  float alpha, beta;
  void *C;
  int64_t ldc;
  int ctype;
  unsigned *dwords;
};

// Instruction descriptor of kind::mxf4: a/b format E2M1 (1 at bits 7-9, 10-11),
// scale type UE8M0 (bit 23), N>>3 at bits 17-22, M>>7 at bits 27-28; the scale
// bytes used (0: the first two, 2: the last two of a TMEM word) at bits 29-30 (A)
// and 4-5 (B).
__device__ __forceinline__ uint32_t idesc_mxf4(int M, int N, uint32_t sf_id) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 7) << 27) |
         (sf_id << 29) | (sf_id << 4);
}

__device__ __forceinline__ void mma_mxf4(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}

// Copies one 512-byte scale tile (32 lines of 16 bytes) to four TMEM columns of
// every lane quarter.
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t saddr) {
  // no swizzle, 8-line groups 128 bytes apart
  const uint64_t desc = (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46);
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          wgtc::smem_addr(dst)),
      "l"(src), "r"(bytes), "r"(wgtc::smem_addr(bar))
      : "memory");
}

struct Tile {
  int g, l0, r0, nv;
  int n_atom;  // scale tile row of the tile's first row
};

template <class S>
__device__ __forceinline__ Tile tile_at(const Args &a, int64_t t, const int *start, const int *tile0,
                                        const int *atom0) {
  Tile x;
  const int q = (int)(t / a.tiles_l);
  x.g = wgg::group_of(tile0, a.groups, q);
  const int ntok = tile0[x.g + 1] - tile0[x.g];
  const int local = (int)(t - (int64_t)tile0[x.g] * a.tiles_l);
  x.l0 = (local / ntok) * BL;
  const int first = (local % ntok) * S::BN;
  x.r0 = start[x.g] + first;
  x.nv = min(S::BN, start[x.g + 1] - x.r0);
  x.n_atom = atom0[x.g] + first / 128;
  return x;
}

template <class S>
__global__ void __launch_bounds__(192, 1)
mx_gemm_kernel(const __grid_constant__ CUtensorMap map_l, const __grid_constant__ CUtensorMap map_n, const Args a) {
  constexpr int STAGES = S::STAGES;
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
  int *tile0 = start + a.groups + 1, *atom0 = tile0 + a.groups + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      wgtc::mbar_init(&full[s], 1);
      wgtc::mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      wgtc::mbar_init(&acc_full[b], 1);
      wgtc::mbar_init(&acc_empty[b], 32 * EPI_WARPS);
    }
    *abort_flag = 0;
    wgtc::fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    wgtc::prefetch_tensormap(&map_l);
    wgtc::prefetch_tensormap(&map_n);
  }
  if (warp == 1) {
    wgtc::tmem_alloc(tmem_slot, S::TMEM_COLS);
    wgtc::tmem_relinquish();
  }
  wg_pdl_wait();
  wg_pdl_trigger();
  wgg::plan_groups(a.offsets, a.groups, a.rows, S::BN, start, tile0, atom0, a.dwords);
  wgtc::tc_fence_before();
  __syncthreads();
  wgtc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int64_t tiles = (int64_t)tile0[a.groups] * a.tiles_l;
  const int kt = a.alpha == 0.0f ? 0 : (a.k + BKE - 1) / BKE;

  if (warp == 0 && lane == 0) {
    // ---- producer: codes by TMA, scale tiles by bulk copies ----
    int64_t it = 0;
    bool ok = true;
    for (int64_t t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const Tile x = tile_at<S>(a, t, start, tile0, atom0);
      const int boxes = (x.nv + 63) / 64, atoms = (x.nv + 127) / 128;
      const uint8_t *sl = a.sf_l + ((int64_t)x.g * a.l_atoms + x.l0 / 128) * a.katoms * 512;
      const uint8_t *sn = a.sf_n + (int64_t)x.n_atom * a.katoms * 512;
      for (int kb = 0; kb < kt; kb++, it++) {
        const int s = (int)(it % STAGES);
        if (!wgtc::mbar_wait_bounded(&empty[s], ((uint32_t)(it / STAGES) & 1u) ^ 1u, WAIT_BUDGET) || *abort_flag) {
          atomicOr(a.dwords + WG_DW_ERROR, WG_DERR_TMA_WAIT);
          *abort_flag = 1;
          ok = false;
          break;
        }
        uint8_t *st = smem + (size_t)s * S::STAGE;
        // The last k-block may have one scale tile instead of two.
        const uint32_t sf = (uint32_t)min(2, a.katoms - kb * 2) * 512u;
        wgtc::mbar_arrive_expect_tx(&full[s], (uint32_t)(S::L_BYTES + boxes * 64 * 128) + sf * (1 + atoms));
        wgtc::tma_load_3d(st, &map_l, &full[s], kb * 128, x.l0, x.g);
        for (int b = 0; b < boxes; b++)
          wgtc::tma_load_2d(st + S::L_BYTES + b * 8192, &map_n, &full[s], kb * 128, x.r0 + b * 64);
        uint8_t *sf_at = st + S::L_BYTES + S::N_BYTES;
        bulk_load(sf_at, sl + kb * 1024, sf, &full[s]);
        for (int b = 0; b < atoms; b++)
          bulk_load(sf_at + 1024 * (1 + b), sn + ((int64_t)b * a.katoms + kb * 2) * 512, sf, &full[s]);
      }
    }
    for (int64_t q = it - STAGES > 0 ? it - STAGES : 0; q < it; q++)
      wgtc::mbar_wait_bounded(&full[q % STAGES], (uint32_t)(q / STAGES) & 1u, WAIT_BUDGET);
  } else if (warp == 1 && lane == 0) {
    // ---- MMA issuer ----
    int64_t it = 0;
    int used = 0;
    bool ok = true;
    for (int64_t t = blockIdx.x; t < tiles && ok && kt; t += gridDim.x, used++) {
      const Tile x = tile_at<S>(a, t, start, tile0, atom0);
      const int nmma = (x.nv + 31) & ~31, atoms = (x.nv + 127) / 128;
      const int b = used % S::ACCS;
      if (!wgtc::mbar_wait_bounded(&acc_empty[b], ((uint32_t)(used / S::ACCS) & 1u) ^ 1u, WAIT_BUDGET) || *abort_flag) {
        atomicOr(a.dwords + WG_DW_ERROR, WG_DERR_MMA_WAIT);
        *abort_flag = 1;
        break;
      }
      wgtc::tc_fence_after();
      const uint32_t d_tmem = tmem + (uint32_t)(b * S::BN);
      for (int kb = 0; kb < kt; kb++, it++) {
        const int s = (int)(it % STAGES);
        if (!wgtc::mbar_wait_bounded(&full[s], (uint32_t)(it / STAGES) & 1u, WAIT_BUDGET) || *abort_flag) {
          atomicOr(a.dwords + WG_DW_ERROR, WG_DERR_TMA_WAIT);
          *abort_flag = 1;
          ok = false;
          break;
        }
        wgtc::tc_fence_after();
        const uint32_t st = wgtc::smem_addr(smem + (size_t)s * S::STAGE);
        const uint32_t sn = st + S::L_BYTES, sf = sn + S::N_BYTES;
        const uint32_t tl = tmem + S::SF_COL + (uint32_t)(it & 1) * S::SF_SET, tn = tl + 8;
        const int katoms = min(2, a.katoms - kb * 2);
        for (int j = 0; j < katoms; j++) {
          copy_scales(tl + 4 * j, sf + 512 * j);
          for (int r = 0; r < atoms; r++) copy_scales(tn + 4 * S::NT * j + 4 * r, sf + 1024 * (1 + r) + 512 * j);
        }
        const int steps = min(4, (a.k - kb * BKE + 63) / 64);
        for (int i = 0; i < steps; i++)
          mma_mxf4(d_tmem, wgtc::smem_desc_kmajor(st + i * 32, 128), wgtc::smem_desc_kmajor(sn + i * 32, 128),
                   idesc_mxf4(BL, nmma, (uint32_t)(i & 1) * 2), tl + 4 * (i >> 1), tn + 4 * S::NT * (i >> 1),
                   (kb > 0 || i > 0) ? 1u : 0u);
        wgtc::mma_commit(&empty[s]);
      }
      if (ok) wgtc::mma_commit(&acc_full[b]);
    }
  } else if (warp >= 2) {
    // ---- epilogue ----
    const int q = warp & 3;
    int used = 0;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x, used++) {
      const Tile x = tile_at<S>(a, t, start, tile0, atom0);
      const int b = used % S::ACCS;
      if (kt) {
        bool ready = wgtc::mbar_wait_bounded(&acc_full[b], (uint32_t)(used / S::ACCS) & 1u, WAIT_BUDGET) && *abort_flag == 0;
        ready = __all_sync(0xffffffffu, ready);
        if (!ready) {
          if (lane == 0) atomicOr(a.dwords + WG_DW_ERROR, WG_DERR_MMA_WAIT);
          *abort_flag = 1;
          break;
        }
        wgtc::tc_fence_after();
      }
      const int l = x.l0 + q * 32 + lane;
      const int64_t at = (int64_t)x.r0 * a.ldc + l;
      const uint32_t trow = tmem + (uint32_t)(b * S::BN) + ((uint32_t)(q * 32) << 16);
      for (int c = 0; c < x.nv; c += 32) {
        uint32_t r[32];
        if (kt) {
          wgtc::tmem_ld_32x32b_x32(trow + (uint32_t)c, r);
          wgtc::tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; j++) r[j] = 0;
        }
        float f[32];
#pragma unroll
        for (int j = 0; j < 32; j++) f[j] = __uint_as_float(r[j]);
        if (l < a.n) wgg::store_cols<32>(a.C, a.ctype, at + (int64_t)c * a.ldc, a.ldc, x.nv - c, a.alpha, a.beta, f);
      }
      wgtc::tc_fence_before();
      mbar_arrive(&acc_empty[b]);
    }
  }

  wgtc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    wgtc::tc_fence_after();
    wgtc::tmem_dealloc(tmem, S::TMEM_COLS);
  }
}

// ---- host side ------------------------------------------------------------

int64_t pitch_of(int64_t cols) { return (cols + 31) / 32 * 16; }
int64_t tiles_of(int64_t n) { return (n + 127) / 128; }

constexpr int64_t LIM = (int64_t)1 << 31;

wg_status check_matrix(const char *name, const void *codes, const void *scales) {
  if (!codes || !scales) return wg_fail(WG_ERR_INVALID_ARGUMENT, "%s: operand pointer is NULL", name);
  if (((uintptr_t)codes & 15) || ((uintptr_t)scales & 15))
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "%s: codes and scales must be 16-byte aligned.", name);
  return WG_OK;
}

wg_status check_quant(const wg_device *d, int type, int64_t batch, int64_t rows, int64_t cols, int64_t groups,
                      const int *offsets) {
  if (!d) return wg_fail(WG_ERR_INVALID_ARGUMENT, "device is NULL");
  if (type != WG_TYPE_F32 && type != WG_TYPE_BF16 && type != WG_TYPE_F16)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "X must be float32, bfloat16 or float16.");
  if (batch < 0 || rows < 0 || cols < 0 || groups < 0)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "batch, rows, cols, and groups must be non-negative.");
  if (rows >= LIM - 1024 || cols >= LIM - 1024)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "dimensions must be below 2^31 - 1024");
  if (groups > WG_MAX_GROUPS)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "groups must be at most %d.", WG_MAX_GROUPS);
  if (groups > 0 && (batch != 1 || !offsets))
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "a matrix with grouped rows has batch 1 and offsets.");
  return WG_OK;
}

wg_status launch_quant(wg_device *d, const char *family, void (*kern)(const QuantArgs), QuantArgs &a) {
  const int64_t tiles = a.offsets ? tiles_of(a.rows) + a.groups : (int64_t)a.batch * a.tiles_r;
  if (tiles * a.tiles_c >= LIM) return wg_fail(WG_ERR_INVALID_ARGUMENT, "too many elements for one call");
  const size_t smem = a.offsets ? 2 * ((size_t)a.groups + 1) * sizeof(int) : 0;
  wg_launch_scope scope(d, family);
  WG_CUDA(wg_launch_pdl(kern, dim3((unsigned)(tiles * a.tiles_c)), dim3(256), smem, d->stream, a));
  WG_CUDA(cudaGetLastError());
  return WG_OK;
}

bool encode(CUtensorMap *map, const void *ptr, int rank, const cuuint64_t *dims, const cuuint64_t *strides,
            const cuuint32_t *box) {
  wg_encode_tiled_fn fn = wg_encode_tiled();
  if (!fn) return false;
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void *>(ptr), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class S>
wg_status launch_gemm(wg_device *d, const char *family, const Args &a, const uint8_t *A, const uint8_t *B) {
  CUtensorMap ml, mn;
  memset(&ml, 0, sizeof ml);
  memset(&mn, 0, sizeof mn);
  if (a.alpha != 0.0f) {
    const cuuint64_t pitch = (cuuint64_t)pitch_of(a.k);
    const cuuint64_t dl[3] = {pitch, (cuuint64_t)a.n, (cuuint64_t)a.groups};
    const cuuint64_t sl[2] = {pitch, pitch * (cuuint64_t)a.n};
    const cuuint32_t bl[3] = {128, (cuuint32_t)BL, 1};
    const cuuint64_t dn[2] = {pitch, (cuuint64_t)a.rows};
    const cuuint32_t bn[2] = {128, 64};
    if (!encode(&ml, B, 3, dl, sl, bl) || !encode(&mn, A, 2, dn, sl, bn))
      return wg_fail(WG_ERR_INVALID_ARGUMENT, "the operands' sizes exceed what a tensor map describes");
  }
  const int64_t most = ((int64_t)a.rows / S::BN + a.groups) * a.tiles_l;
  const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(most, d->sm_count));
  wg_launch_scope scope(d, family);
  WG_CUDA(wg_kernel_smem(mx_gemm_kernel<S>, SMEM_LIMIT));
  WG_CUDA(wg_launch_pdl(mx_gemm_kernel<S>, dim3(grid), dim3(192), S::smem(a.groups), d->stream, ml, mn, a));
  WG_CUDA(cudaGetLastError());
  return WG_OK;
}

wg_status mx_gemm(wg_device *d, const char *family, int ctype, int64_t groups, int64_t m, int64_t n, int64_t k,
                  float alpha, const void *A, const void *As, const void *B, const void *Bs, const int *offsets,
                  float beta, void *C, int64_t ldc, float *gpu_ms) {
  if (gpu_ms) *gpu_ms = 0.0f;
  if (!d) return wg_fail(WG_ERR_INVALID_ARGUMENT, "device is NULL");
  if (ctype != WG_TYPE_F32 && ctype != WG_TYPE_BF16 && ctype != WG_TYPE_F16)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "C must be float32, bfloat16 or float16.");
  if (groups < 0 || m < 0 || n < 0 || k < 0)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "groups, m, n, and k must be non-negative.");
  if (groups > WG_MAX_GROUPS)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "groups must be at most %d.", WG_MAX_GROUPS);
  if (m >= LIM - 1024 || n >= LIM - 1024 || k >= LIM - 1024)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "dimensions must be below 2^31 - 1024");
  if (ldc <= 0) return wg_fail(WG_ERR_INVALID_ARGUMENT, "ldc must be positive.");
  if (ldc < n) return wg_fail(WG_ERR_INVALID_ARGUMENT, "ldc must be >= cols of C as stored.");
  if (ldc >= ((int64_t)1 << 40)) return wg_fail(WG_ERR_INVALID_ARGUMENT, "leading dimensions must be below 2^40");
  if (groups == 0 || m == 0 || n == 0) return WG_OK;
  if (!C) return wg_fail(WG_ERR_INVALID_ARGUMENT, "operand pointer is NULL");
  if (k == 0) alpha = 0.0f;
  wg_status st;
  if (alpha != 0.0f && ((st = check_matrix("A", A, As)) != WG_OK || (st = check_matrix("B", B, Bs)) != WG_OK)) return st;
  st = wgg::check_arch(d);
  if (st != WG_OK) return st;
  if (alpha == 0.0f && beta == 1.0f) return WG_OK;  // C stays as it is
  wg_device_guard guard(d->ordinal);
  Args a = {};
  a.groups = (int)groups;
  a.rows = (int)m;
  a.n = (int)n;
  a.k = (int)k;
  a.tiles_l = (int)tiles_of(n);
  a.katoms = (int)tiles_of(k);
  a.l_atoms = (int)tiles_of(n);
  a.offsets = offsets;
  a.sf_l = static_cast<const uint8_t *>(Bs);
  a.sf_n = static_cast<const uint8_t *>(As);
  a.alpha = alpha;
  a.beta = beta;
  a.C = C;
  a.ldc = ldc;
  a.ctype = ctype;
  a.dwords = d->dwords;
  const uint8_t *pa = static_cast<const uint8_t *>(A), *pb = static_cast<const uint8_t *>(B);
  return wg_timed(d, gpu_ms, [&] {
    return m / groups <= 128 ? launch_gemm<Shape<128>>(d, family, a, pa, pb)
                             : launch_gemm<Shape<256>>(d, family, a, pa, pb);
  });
}

}  // namespace

extern "C" wg_status wg_mx_quantize_dev(wg_device *d, int type, int trans, int64_t batch, int64_t rows, int64_t cols,
                                        const void *X, int64_t ldx, int64_t strideX, int64_t groups,
                                        const int *offsets, void *codes, void *scales, float *gpu_ms) {
  if (gpu_ms) *gpu_ms = 0.0f;
  wg_status st = check_quant(d, type, batch, rows, cols, groups, offsets);
  if (st != WG_OK) return st;
  if (trans != 0 && trans != 1)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "trans must be 'no-transpose' or 'transpose'.");
  if (trans && groups) return wg_fail(WG_ERR_INVALID_ARGUMENT, "grouped rows are quantised without transpose.");
  if (ldx <= 0 || ldx >= ((int64_t)1 << 40) || strideX < 0 || strideX >= ((int64_t)1 << 40))
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "ldx must be positive, strideX non-negative, both below 2^40.");
  if (ldx < (trans ? rows : cols)) return wg_fail(WG_ERR_INVALID_ARGUMENT, "ldx must be >= cols of X as stored.");
  if (batch == 0 || rows == 0 || cols == 0) return WG_OK;
  if (!X) return wg_fail(WG_ERR_INVALID_ARGUMENT, "operand pointer is NULL");
  if ((st = check_matrix("out", codes, scales)) != WG_OK || (st = wgg::check_arch(d)) != WG_OK) return st;
  if (batch >= LIM || batch * tiles_of(rows) >= LIM) return wg_fail(WG_ERR_INVALID_ARGUMENT, "too many elements for one call");
  wg_device_guard guard(d->ordinal);
  QuantArgs a = {X, ldx, strideX, type, (int)rows, (int)cols, static_cast<uint8_t *>(codes),
                 static_cast<uint8_t *>(scales), pitch_of(cols), (int)tiles_of(rows), (int)tiles_of(cols), (int)batch,
                 groups ? offsets : nullptr, (int)groups, d->dwords};
  return wg_timed(d, gpu_ms, [&] {
    void (*kern)(const QuantArgs);
    if (trans)
      kern = type == WG_TYPE_F32 ? mx_quantize_t<float> : type == WG_TYPE_BF16 ? mx_quantize_t<__nv_bfloat16> : mx_quantize_t<__half>;
    else
      kern = type == WG_TYPE_F32 ? mx_quantize<float> : type == WG_TYPE_BF16 ? mx_quantize<__nv_bfloat16> : mx_quantize<__half>;
    return launch_quant(d, "mx_quantize", kern, a);
  });
}

extern "C" wg_status wg_mx_dequantize_dev(wg_device *d, int type, int64_t batch, int64_t rows, int64_t cols,
                                          const void *codes, const void *scales, int64_t groups, const int *offsets,
                                          void *X, int64_t ldx, int64_t strideX, float *gpu_ms) {
  if (gpu_ms) *gpu_ms = 0.0f;
  wg_status st = check_quant(d, type, batch, rows, cols, groups, offsets);
  if (st != WG_OK) return st;
  if (ldx <= 0 || ldx >= ((int64_t)1 << 40) || strideX < 0 || strideX >= ((int64_t)1 << 40))
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "ldx must be positive, strideX non-negative, both below 2^40.");
  if (ldx < cols) return wg_fail(WG_ERR_INVALID_ARGUMENT, "ldx must be >= cols of X as stored.");
  if (batch > 1 && rows > 0 && strideX < (rows - 1) * ldx + cols)
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "strideX must be at least one matrix of X.");
  if (batch == 0 || rows == 0 || cols == 0) return WG_OK;
  if (!X) return wg_fail(WG_ERR_INVALID_ARGUMENT, "operand pointer is NULL");
  if ((st = check_matrix("X", codes, scales)) != WG_OK || (st = wgg::check_arch(d)) != WG_OK) return st;
  if (batch >= LIM || batch * tiles_of(rows) >= LIM) return wg_fail(WG_ERR_INVALID_ARGUMENT, "too many elements for one call");
  wg_device_guard guard(d->ordinal);
  QuantArgs a = {X, ldx, strideX, type, (int)rows, (int)cols, static_cast<uint8_t *>(const_cast<void *>(codes)),
                 static_cast<uint8_t *>(const_cast<void *>(scales)), pitch_of(cols), (int)tiles_of(rows),
                 (int)tiles_of(cols), (int)batch, groups ? offsets : nullptr, (int)groups, d->dwords};
  return wg_timed(d, gpu_ms, [&] {
    return launch_quant(d, "mx_dequantize",
                        type == WG_TYPE_F32 ? mx_dequantize<float>
                        : type == WG_TYPE_BF16 ? mx_dequantize<__nv_bfloat16> : mx_dequantize<__half>, a);
  });
}

extern "C" wg_status wg_mx_gemm_dev(wg_device *d, int ctype, int64_t m, int64_t n, int64_t k, float alpha,
                                    const void *A, const void *A_scales, const void *B, const void *B_scales,
                                    float beta, void *C, int64_t ldc, float *gpu_ms) {
  return mx_gemm(d, "mx_gemm", ctype, 1, m, n, k, alpha, A, A_scales, B, B_scales, nullptr, beta, C, ldc, gpu_ms);
}

extern "C" wg_status wg_mx_gemm_grouped_dev(wg_device *d, int ctype, int64_t groups, int64_t m, int64_t n, int64_t k,
                                            float alpha, const void *A, const void *A_scales, const void *B,
                                            const void *B_scales, const int *offsets, float beta, void *C, int64_t ldc,
                                            float *gpu_ms) {
  if (gpu_ms) *gpu_ms = 0.0f;
  if (groups > 0 && !offsets) return wg_fail(WG_ERR_INVALID_ARGUMENT, "operand pointer is NULL");
  return mx_gemm(d, "mx_gemm_grouped", ctype, groups, m, n, k, alpha, A, A_scales, B, B_scales, offsets, beta, C, ldc,
                 gpu_ms);
}
