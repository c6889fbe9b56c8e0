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
#include <type_traits>

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

// Eight elements as they are stored.
template <class T>
union Eight {
  uint4 w[sizeof(T) / 2];
  T v[8];
  __device__ __forceinline__ Eight() {}
};

// The float32 bits of the largest magnitude of eight elements (a NaN is larger
// than any number). 16-bit types compare as pairs of integers.
__device__ __forceinline__ uint32_t top_of(const Eight<float> &w) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(w.v[i]) & 0x7fffffffu);
  return top;
}
template <class T>
__device__ __forceinline__ uint32_t top_of(const Eight<T> &w) {
  const uint4 u = w.w[0];
  const uint32_t m = 0x7fff7fffu;
  const uint32_t p = __vmaxu2(__vmaxu2(u.x & m, u.y & m), __vmaxu2(u.z & m, u.w & m));
  const uint16_t h = (uint16_t)max(p & 0xffffu, p >> 16);
  return __float_as_uint(to_float(*reinterpret_cast<const T *>(&h)));
}

// Eight elements at p, of which the first `valid` exist (zeros instead of the
// others), at any alignment: the 16-byte units that hold them, shifted into place
// by words and half words. Memory outside [lo, hi) is not read.
template <class T>
__device__ __forceinline__ void load_eight(Eight<T> &out, const T *p, int valid, const T *lo, const T *hi) {
  constexpr int U = sizeof(T) / 2 + 1, WORDS = 4 * (U - 1);
  const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15;
  const T *base = p - off / sizeof(T);
  if (valid > 0 && base >= lo && base + U * 16 / sizeof(T) <= hi) {
    uint32_t w[4 * U];
#pragma unroll
    for (int i = 0; i < U; i++) {
      const uint4 v = __ldg(reinterpret_cast<const uint4 *>(base) + i);
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
    if (off & 4)
#pragma unroll
      for (int i = 0; i < WORDS + 3; i++) w[i] = w[i + 1];
    if (off & 8)
#pragma unroll
      for (int i = 0; i < WORDS + 1; i++) w[i] = w[i + 2];
    uint32_t x[WORDS];
#pragma unroll
    for (int i = 0; i < WORDS; i++) x[i] = sizeof(T) == 2 ? __funnelshift_r(w[i], w[i + 1], (off & 2) * 8) : w[i];
#pragma unroll
    for (int i = 0; i < WORDS / 4; i++) out.w[i] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i >= valid) out.v[i] = T(0.0f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) out.v[i] = i < valid ? p[i] : T(0.0f);
  }
}

// The rows of one scale tile: first row, how many, and its matrix (batch).
struct TileRows {
  int r0, n, b;
};
// Grouped matrices: every warp finds its tile's group by itself, 32 groups at a
// time, from the same clamped, non-decreasing offsets as plan_groups makes (the
// first CTA goes through them all and reports offsets that this changes).
__device__ __forceinline__ TileRows grouped_rows(const QuantArgs &a, int tile) {
  const int lane = threadIdx.x & 31;
  const bool check = blockIdx.x == 0 && threadIdx.x < 32;
  TileRows t = {0, 0, 0};
  const int first = a.offsets[0];
  int top = max(min(first, a.rows), 0), tiles = 0;
  bool bad = first != top, found = false;
  for (int base = 0; base < a.groups && (!found || check); base += 32) {
    const int j = base + lane;
    const int raw = j < a.groups ? a.offsets[j + 1] : 0;
    int end = max(min(raw, a.rows), 0);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, end, d);
      if (lane >= d) end = max(end, o);
    }
    end = max(end, top);
    bad |= j < a.groups && end != raw;
    int start = __shfl_up_sync(0xffffffffu, end, 1);
    if (lane == 0) start = top;
    const int mine = (end - start + 127) >> 7;  // (0 past the last group: end stays)
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    sum += tiles;
    const uint32_t hit = __ballot_sync(0xffffffffu, tile < sum);
    if (hit && !found) {
      const int f = __ffs(hit) - 1;
      const int s0 = __shfl_sync(0xffffffffu, start, f), e0 = __shfl_sync(0xffffffffu, end, f);
      t.r0 = s0 + (tile - __shfl_sync(0xffffffffu, sum - mine, f)) * 128;
      t.n = min(128, e0 - t.r0);
      found = true;
    }
    top = __shfl_sync(0xffffffffu, end, 31);
    tiles = __shfl_sync(0xffffffffu, sum, 31);
  }
  if (check && bad) atomicOr(a.dwords + WG_DW_ERROR, WG_DERR_OFFSETS);
  return t;
}
__device__ __forceinline__ TileRows rows_of_tile(const QuantArgs &a, int tile) {
  if (a.offsets) return grouped_rows(a, tile);
  TileRows t;
  t.b = tile / a.tiles_r;
  t.r0 = (tile - t.b * a.tiles_r) * 128;
  t.n = min(128, a.rows - t.r0);
  return t;
}

// Scales of two neighbouring tiles (128 rows x 256 columns) of a tile row,
// between shared memory and their place.
__device__ __forceinline__ uint32_t *tile_scales(const QuantArgs &a, int tile, int tc) {
  return reinterpret_cast<uint32_t *>(a.scales + ((int64_t)tile * a.tiles_c + tc) * 512);
}
__device__ __forceinline__ int scale_at(int r, int block) {  // block 0 .. 7 of the two tiles
  return (block >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (block & 3);
}

// A CTA's part of the matrix: two neighbouring scale tiles, of whose rows it takes
// all (STEP 8: its warps take one line in eight), or a quarter (STEP 32: a warp takes
// lines r0 + warp, 32 apart, four in all, whose scales are neighbours too).
struct Part {
  int tile, tc, r0;
};
template <int STEP>
__device__ __forceinline__ Part part_of(const QuantArgs &a) {
  const unsigned pairs = (unsigned)(a.tiles_c + 1) >> 1, x = STEP == 32 ? blockIdx.x >> 2 : blockIdx.x;
  return {(int)(x / pairs), (int)(x % pairs) * 2, STEP == 32 ? (int)(blockIdx.x & 3) * 8 : 0};
}
// Elements from a matrix's first to its last (stored rows x cols).
__device__ __forceinline__ int64_t used_elements(const QuantArgs &a) { return (int64_t)(a.rows - 1) * a.ldx + a.cols; }

constexpr int ROWS_AT_ONCE = 4;  // a warp's loads in flight

// A CTA per part (launch_rows): a warp takes whole 256-column lines, eight
// elements a thread, four threads a block. Bound by memory: 16-byte loads, four
// in flight a thread; a line's codes are one 128-byte store, the scales are
// gathered in shared memory and written as one piece. 8192 x 8192 bf16: 32 us, 5.3
// TB/s of reads and writes (a copy's rate here is 6.55); back, 33 us. Sixteen threads a
// line and one line in flight a thread took 54 and 65 us.
template <class T, int STEP>
__global__ void __launch_bounds__(256) mx_quantize(const QuantArgs a) {
  __shared__ __align__(16) uint8_t sf[1024];
  wg_pdl_wait();
  wg_pdl_trigger();
  const Part part = part_of<STEP>(a);
  const int tile = part.tile, tc = part.tc;
  const TileRows t = rows_of_tile(a, tile);
  if (t.n <= 0) return;
  reinterpret_cast<uint32_t *>(sf)[threadIdx.x] = 0;
  __syncthreads();
  const int warp = threadIdx.x >> 5, c = threadIdx.x & 31, col = tc * 128 + c * 8;
  const T *X = static_cast<const T *>(a.X) + t.b * a.strideX + col;
  const bool in = col / 32 * 16 < a.pitch;  // the block exists (it may end in padding)
  const int valid = in ? a.cols - col : 0;
  // (the whole warp takes one way: the lines' shuffles need all its lanes)
  const bool wide = __all_sync(0xffffffffu, valid >= 8 && ((uintptr_t)X & 15) == 0 && a.ldx * sizeof(T) % 16 == 0);
  uint8_t *codes = a.codes + (int64_t)t.b * a.rows * a.pitch + col / 2;
  int r = part.r0 + warp;
  const T *src = X + (t.r0 + (int64_t)r) * a.ldx;
  uint8_t *dst = codes + (t.r0 + (int64_t)r) * a.pitch;
  const T *lo = static_cast<const T *>(a.X) + t.b * a.strideX, *hi = lo + used_elements(a);
  uint8_t *sfb = sf + (c >> 4) * 512 + (c >> 2 & 3);
  const int64_t src_step = STEP * a.ldx, dst_step = STEP * a.pitch;
  // Rounds one line's eight elements; `r` is the line within the tile.
  auto round = [&](const Eight<T> &w, uint8_t *to, int r) {
    uint32_t top = top_of(w);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t e = scale_byte(top);
    const float inv = inverse_scale(e);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = to_float(w.v[i]) * inv;
    if (in) {
      *reinterpret_cast<uint32_t *>(to) = encode8(x);
      if ((c & 3) == 0) sfb[(r & 31) * 16 + (r >> 5) * 4] = (uint8_t)e;
    }
  };
  // Lines past the end are read as the last one, so that a batch's loads go out
  // together whatever its length.
  auto batch = [&](auto count, int r, const T *from, uint8_t *to) {
    constexpr int N = decltype(count)::value;
    Eight<T> w[N];
    const int last = (t.n - 1 - r) / STEP;
#pragma unroll
    for (int u = 0; u < N; u++) {
      const T *p = from + min(u, last) * src_step;
      if (wide) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) w[u].w[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
      } else {
        load_eight(w[u], p, valid, lo, hi);
      }
    }
#pragma unroll
    for (int u = 0; u < N; u++)
      if (u <= last) round(w[u], to + u * dst_step, r + STEP * u);
  };
  if constexpr (STEP == 32) {
    if (r < t.n) batch(std::integral_constant<int, 4>(), r, src, dst);
  } else {
    if (wide && t.n > 64)
      for (; r + 8 * (ROWS_AT_ONCE - 1) < t.n; r += 8 * ROWS_AT_ONCE) {
        Eight<T> w[ROWS_AT_ONCE];
#pragma unroll
        for (int u = 0; u < ROWS_AT_ONCE; u++, src += src_step)
#pragma unroll
          for (int i = 0; i < (int)sizeof(T) / 2; i++) w[u].w[i] = __ldg(reinterpret_cast<const uint4 *>(src) + i);
#pragma unroll
        for (int u = 0; u < ROWS_AT_ONCE; u++, dst += dst_step) round(w[u], dst, r + 8 * u);
      }
    // The rest (all of a short tile, at once), and lines that wide loads cannot read.
    constexpr int REST = 8;
    for (; r < t.n; r += 8 * REST, src += REST * src_step, dst += REST * dst_step)
      batch(std::integral_constant<int, REST>(), r, src, dst);
  }
  __syncthreads();
  // (the second tile exists unless the tile row has an odd number of them)
  constexpr int WORDS = STEP == 32 ? 32 : 128;
  if (threadIdx.x < WORDS || (threadIdx.x < 2 * WORDS && tc + 1 < a.tiles_c)) {
    const int i = (int)(threadIdx.x / WORDS) * 128 + part.r0 * 4 + (int)(threadIdx.x % WORDS);
    tile_scales(a, tile, tc)[i] = reinterpret_cast<const uint32_t *>(sf)[i];
  }
}

// The transposed form: X holds the matrix's columns as its rows. One CTA per
// scale tile; a thread takes two neighbouring rows of the result and one block
// of them, 32 of X's lines: its loads are independent, and a warp's are 64
// neighbouring elements. The codes go through shared memory, so that a row's four
// blocks are stored together (8192 x 8192 bf16: 34.5 us, with each thread's 16 bytes
// stored on their own 38.2).
template <class T>
struct Two {
  T v[2];
};
template <class T>
__global__ void __launch_bounds__(256) mx_quantize_t(const QuantArgs a) {
  __shared__ __align__(16) uint8_t sf[512];
  __shared__ uint4 out[128 * 5];  // the tile's codes, four blocks a row (and one for the banks)
  wg_pdl_wait();
  wg_pdl_trigger();
  const int tile = (int)(blockIdx.x / (unsigned)a.tiles_c), tc = (int)(blockIdx.x % (unsigned)a.tiles_c);
  const TileRows t = rows_of_tile(a, tile);
  if (threadIdx.x < 128) reinterpret_cast<uint32_t *>(sf)[threadIdx.x] = 0;
  __syncthreads();
  const int blk = threadIdx.x >> 6, r = (threadIdx.x & 63) * 2, col = tc * 128 + blk * 32;
  if (r < t.n && col / 32 * 16 < a.pitch) {
    const T *X = static_cast<const T *>(a.X) + t.b * a.strideX + (int64_t)col * a.ldx + t.r0 + r;
    const int valid = a.cols - col;
    const bool both = r + 1 < t.n;
    Two<T> w[32];
    if (both && valid >= 32 && ((uintptr_t)X % sizeof(Two<T>)) == 0 && a.ldx % 2 == 0) {
#pragma unroll
      for (int i = 0; i < 32; i++) {
        if constexpr (sizeof(T) == 2) {
          const uint32_t v = __ldg(reinterpret_cast<const uint32_t *>(X + i * a.ldx));
          w[i] = *reinterpret_cast<const Two<T> *>(&v);
        } else {
          const uint2 v = __ldg(reinterpret_cast<const uint2 *>(X + i * a.ldx));
          w[i] = *reinterpret_cast<const Two<T> *>(&v);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; i++) {
        w[i].v[0] = i < valid ? X[i * a.ldx] : T(0.0f);
        w[i].v[1] = i < valid && both ? X[i * a.ldx + 1] : T(0.0f);
      }
    }
#pragma unroll
    for (int p = 0; p < 2; p++) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 32; i++) top = max(top, __float_as_uint(to_float(w[i].v[p])) & 0x7fffffffu);
      const uint32_t e = scale_byte(top);
      const float inv = inverse_scale(e);
      uint32_t code[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float y[8];
#pragma unroll
        for (int k = 0; k < 8; k++) y[k] = to_float(w[i * 8 + k].v[p]) * inv;
        code[i] = encode8(y);
      }
      if (p == 0 || both) {
        out[(r + p) * 5 + blk] = make_uint4(code[0], code[1], code[2], code[3]);
        sf[scale_at(r + p, blk)] = (uint8_t)e;
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < t.n * 4; i += 256) {
    const int row = i >> 2, b = i & 3;
    const int64_t at = tc * 64 + b * 16;
    if (at < a.pitch)
      *reinterpret_cast<uint4 *>(a.codes + ((int64_t)t.b * a.rows + t.r0 + row) * a.pitch + at) = out[row * 5 + b];
  }
  if (threadIdx.x < 128) tile_scales(a, tile, tc)[threadIdx.x] = reinterpret_cast<const uint32_t *>(sf)[threadIdx.x];
}

// ---- the values the codes stand for ------------------------------------------

template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// Four codes' values. An element's bits moved to the low end of an fp16's exponent
// field and the top of its mantissa are the element times 2^-14 (its exponent bias
// is 1, fp16's 15; subnormals stay subnormal); every product below is exact.
__device__ __forceinline__ void decode4(uint32_t code, float scale, float *y) {
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint32_t b = code >> (8 * i);
    const uint32_t h = (b & 0x07u) << 9 | (b & 0x08u) << 12 | (b & 0x70u) << 21 | (b & 0x80u) << 24;
    const float2 f = __half22float2(__hmul2(*reinterpret_cast<const __half2 *>(&h), __float2half2_rn(16384.0f)));
    y[2 * i] = f.x * scale;
    y[2 * i + 1] = f.y * scale;
  }
}

// X here is the output (rows x cols, ldx), of rows of whole 16-byte units. The
// quantiser's division of the work; a thread's store is 16 bytes, a warp's 512
// neighbouring ones (an fp32 line takes two). Whole tile pairs load eight lines of codes
// at once (4096 x 4096 bf16: 9.1 us, four at once 12.9).
template <class T, int STEP>
__global__ void __launch_bounds__(256) mx_dequantize(const QuantArgs a) {
  constexpr int E = 16 / sizeof(T), PASSES = 8 / E, AT_ONCE = STEP == 8 ? 8 : 4;
  __shared__ __align__(16) uint8_t sf[1024];
  wg_pdl_wait();
  wg_pdl_trigger();
  const Part part = part_of<STEP>(a);
  const int tile = part.tile, tc = part.tc;
  const TileRows t = rows_of_tile(a, tile);
  if (t.n <= 0) return;
  if (threadIdx.x < 128 || tc + 1 < a.tiles_c) reinterpret_cast<uint32_t *>(sf)[threadIdx.x] = tile_scales(a, tile, tc)[threadIdx.x];
  __syncthreads();
  const int c = threadIdx.x & 31, first = part.r0 + (int)(threadIdx.x >> 5);
  T *X = static_cast<T *>(const_cast<void *>(a.X)) + t.b * a.strideX;
  const uint8_t *codes = a.codes + (int64_t)t.b * a.rows * a.pitch;
#pragma unroll
  for (int p = 0; p < PASSES; p++) {
    const int in_tiles = p * 32 * E + c * E, col = tc * 128 + in_tiles;
    if (col >= a.cols) return;
    const uint8_t *src = codes + (t.r0 + (int64_t)first) * a.pitch + col / 2;
    T *dst = X + (t.r0 + (int64_t)first) * a.ldx + col;
    const uint8_t *sfb = sf + scale_at(0, in_tiles >> 5);
    const int64_t src_step = STEP * a.pitch, dst_step = STEP * a.ldx;
    const bool wide = col + E <= a.cols;
    auto load = [&](const uint8_t *at) -> uint32_t {
      if constexpr (E == 8) return __ldg(reinterpret_cast<const uint32_t *>(at));
      else return __ldg(reinterpret_cast<const uint16_t *>(at));
    };
    auto store = [&](uint32_t code, T *to, int r) {
      const float s = scale_value(sfb[(r & 31) * 16 + (r >> 5) * 4]);
      float f[E];
#pragma unroll
      for (int i = 0; i < E / 4; i++) decode4(code >> (16 * i), s, f + 4 * i);
      alignas(16) T y[E];
#pragma unroll
      for (int i = 0; i < E; i++) y[i] = from_float<T>(f[i]);
      if (wide) {
        *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(y);
      } else {
#pragma unroll
        for (int i = 0; i < E; i++)
          if (col + i < a.cols) to[i] = y[i];
      }
    };
    int r = first;
    for (; r + STEP * (AT_ONCE - 1) < t.n; r += STEP * AT_ONCE) {
      uint32_t code[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; u++, src += src_step) code[u] = load(src);
#pragma unroll
      for (int u = 0; u < AT_ONCE; u++, dst += dst_step) store(code[u], dst, r + STEP * u);
    }
    if (r < t.n) {
      const int last = (t.n - 1 - r) / STEP;
      uint32_t code[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; u++) code[u] = load(src + min(u, last) * src_step);
#pragma unroll
      for (int u = 0; u < AT_ONCE; u++)
        if (u <= last) store(code[u], dst + u * dst_step, r + STEP * u);
    }
  }
}

// Rows of any alignment: lane c stores elements c, c + 32, ... of a line, so that a
// warp's store is 32 neighbouring ones; their codes are in words of other lanes.
// (16-byte-aligned threads storing element by element: 8001 x 8001 bf16 183 us, this 63.)
template <class T>
__global__ void __launch_bounds__(256) mx_dequantize_unaligned(const QuantArgs a) {
  __shared__ __align__(16) uint8_t sf[1024];
  wg_pdl_wait();
  wg_pdl_trigger();
  const Part part = part_of<32>(a);
  const int tile = part.tile, tc = part.tc;
  const TileRows t = rows_of_tile(a, tile);
  if (t.n <= 0) return;
  if (threadIdx.x < 128 || tc + 1 < a.tiles_c) reinterpret_cast<uint32_t *>(sf)[threadIdx.x] = tile_scales(a, tile, tc)[threadIdx.x];
  __syncthreads();
  const int c = threadIdx.x & 31, first = part.r0 + (int)(threadIdx.x >> 5);
  T *X = static_cast<T *>(const_cast<void *>(a.X)) + t.b * a.strideX;
  const uint8_t *codes = a.codes + (int64_t)t.b * a.rows * a.pitch;
  const bool in = tc * 128 + c * 8 < ((a.cols + 31) & ~31);  // this lane's word of codes exists
  uint32_t word[4];
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const int r = first + 32 * u;
    word[u] = in && r < t.n ? __ldg(reinterpret_cast<const uint32_t *>(codes + (t.r0 + (int64_t)r) * a.pitch) + tc * 16 + c) : 0;
  }
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const int r = first + 32 * u;
    T *to = X + (t.r0 + (int64_t)r) * a.ldx + tc * 128 + c;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      float f[4];
      decode4(__shfl_sync(0xffffffffu, word[u], 4 * i + (c >> 3)) >> (4 * (c & 7)) & 15u, scale_value(sf[scale_at(r, i)]), f);
      if (r < t.n && tc * 128 + i * 32 + c < a.cols) to[i * 32] = from_float<T>(f[0]);
    }
  }
}

// ---- product ------------------------------------------------------------------
//
// The grouped kernel's frame and roles (grouped.cu): B's rows on the lanes, A's
// rows on the columns, both K-major. A k-block is 256 elements, 128 bytes of
// codes a row and two scale tiles for each 128 rows of an operand; the MMA warp
// copies the scale tiles to TMEM (tcgen05.cp, four columns a tile) in front of
// the block's four MMAs of 64.
//
// Forms: CTA pairs with 256 x 256 tiles for compute-bound calls (an MMA of 64
// takes as long as a bf16 one of 16, so the bytes a tile needs from L2 a clock
// are the same as there, and with them the reason for pairs), one CTA with
// 128 columns otherwise, or a cluster of such that splits the contraction; 32
// columns where the call has no more rows. (Tiles begin at whole scale tiles, 128
// rows, of their group: the address of an MMA's scales in TMEM cannot be any
// column. 32-column tiles inside a scale tile, at an odd one, raised "misaligned
// address".) A pair's accumulator and scales leave no room for a
// second accumulator in TMEM: the epilogue drains it to registers at once and
// stores from there while the next tile's MMAs run.

constexpr int BKE = 256;           // elements of a k-block
constexpr int EPI_WARPS = wgg::EPI_WARPS;
constexpr size_t SMEM_LIMIT = 227 * 1024;
// k-blocks between drains of the accumulator, whose additions truncate (grouped.cu): up
// to 3e-10 of the sum a contraction row here (measured at 2^19 rows, positive values over
// many powers of two; sums of values alike are exact for longer). SEG: fp32 results and
// split contractions. LONG: 16-bit results, 65536 rows, 1024 MMAs that lose at most 2^-23 of a
// partial sum each, 6.1e-5 of the whole: an eighth of fp16's half step (2^-11). bf16's
// (2^-8) is eight times that, so its sums are drained beyond 524288 rows only.
constexpr int SEG = 16, LONG = 256;
// Rows of a 16-bit result's contraction that one accumulator takes whole.
constexpr int whole_rows(int type) { return type == WG_TYPE_BF16 ? 8 * LONG * BKE : LONG * BKE; }

// CG CTAs (a pair or one) share a tile's lanes, P CTAs its contraction.
template <int CG_, int BN_, int P_ = 1>
struct Shape {
  static constexpr int CG = CG_, BN = BN_, P = P_, CLUSTER = CG * P;
  static_assert(CG == 1 || P == 1, "a pair shares lanes or contraction, not both");
  static constexpr int TL = CG * BL, CPT = BN / 2;
  static constexpr int NT = BN > 128 ? BN / 128 : 1;  // scale tiles of the N side (every CTA of a pair has all)
  static constexpr int NBOX = BN < 64 ? BN : 64;      // rows of one N-side box
  static constexpr int L_BYTES = BL * 128, N_BYTES = BN / CG * 128;
  static constexpr int SF_L = 1024, SF_N = NT * 1024;
  static constexpr int STAGE = L_BYTES + N_BYTES + SF_L + SF_N;
  static constexpr int PARTS = (P - 1) * BN * BL * 4;
  static constexpr int STAGES = (int)((SMEM_LIMIT - 14 * 1024 - PARTS) / STAGE);
  // TMEM columns: accumulators, then two sets of scales (L: 2 x 4, N: 2 x 4 NT).
  static constexpr int ACCS = BN <= 128 ? 2 : 1;
  static constexpr int SF_COL = ACCS * BN, SF_SET = 8 + 8 * NT;
  static constexpr int TMEM_COLS = BN <= 32 ? 128 : 512;
  static_assert(BN == 32 || BN % 128 == 0, "tiles begin at whole scale tiles");
  static_assert(SF_COL + 2 * SF_SET <= TMEM_COLS, "accumulators and scales must fit TMEM");
  static constexpr size_t parts = (size_t)STAGES * STAGE;
  static constexpr size_t bars = parts + PARTS;
  static constexpr size_t tables = bars + 256;
  static constexpr size_t smem(int groups) { return 1024 + tables + 3 * ((size_t)groups + 1) * sizeof(int); }
  static constexpr int NMMA_STEP = 32;
};

struct Args {
  int groups, rows, n, k;
  int tiles_l;
  int l_atoms;           // scale tile rows of one matrix of B
  const int *offsets;    // NULL: one group, all rows
  wgg::Out out;
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

template <int CG>
__device__ __forceinline__ void mma_mxf4(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// Copies one 512-byte scale tile (32 lines of 16 bytes, no swizzle, eight-line
// groups 128 bytes apart) to four TMEM columns of every lane quarter; for a pair,
// each CTA from its own shared memory to its own TMEM.
__device__ __forceinline__ uint64_t scales_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46);
}
template <int CG>
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

struct Tile {
  int g, l0, r0, nv;
  int n_atom;  // scale tile row of the tile's first row
  int k_lo, k_hi;  // this CTA's k-blocks
};

template <class S>
__device__ __forceinline__ Tile tile_at(const Args &a, int64_t t, const int *start, const int *tile0,
                                        const int *atom0, int kt, uint32_t rank) {
  Tile x;
  const int q = (int)(t / a.tiles_l);
  x.g = wgg::group_of(tile0, a.groups, q);
  const int ntok = tile0[x.g + 1] - tile0[x.g];
  const int local = (int)(t - (int64_t)tile0[x.g] * a.tiles_l);
  x.l0 = (local / ntok) * S::TL;
  const int first = (local % ntok) * S::BN;
  x.r0 = start[x.g] + first;
  x.nv = min(S::BN, start[x.g + 1] - x.r0);
  x.n_atom = atom0[x.g] + first / 128;
  x.k_lo = S::P > 1 ? (int)((int64_t)kt * rank / S::P) : 0;
  x.k_hi = S::P > 1 ? (int)((int64_t)kt * (rank + 1) / S::P) : kt;
  return x;
}

// Warps: 0 and 10 load (the L and the N side, codes and scales), 1 issues the
// MMAs, 2-9 store. DRAIN: k-blocks after which the accumulator is drained (SEG, LONG; 0:
// at the tile's end).
template <class S, int DRAIN>
__global__ void __launch_bounds__(352, 1)
mx_gemm_kernel(const __grid_constant__ CUtensorMap map_l, const __grid_constant__ CUtensorMap map_n,
               const __grid_constant__ CUtensorMap map_sl, const __grid_constant__ CUtensorMap map_sn, const Args a) {
  constexpr int STAGES = S::STAGES, CG = S::CG;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = wgtc::smem_addr(smem_raw);
  uint8_t *smem = smem_raw + ((1024 - (base & 1023)) & 1023);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + S::bars);
  uint64_t *empty = full + STAGES;
  uint64_t *acc_full = empty + STAGES;  // [2]
  uint64_t *acc_empty = acc_full + 2;   // [2]
  wgg::Parts parts = {reinterpret_cast<float *>(smem + S::parts), acc_empty + 2, acc_empty + 3, 0};
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 4);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  int *start = reinterpret_cast<int *>(smem + S::tables);
  int *tile0 = start + a.groups + 1, *atom0 = tile0 + a.groups + 1;

  const int warp = wgg::warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = S::CLUSTER > 1 ? wgtc::cluster_ctarank() : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      wgtc::mbar_init(&full[s], 2);
      wgtc::mbar_init(&empty[s], 1);
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
  if (warp == 0 && lane == 0) {
    wgtc::prefetch_tensormap(&map_l);
    wgtc::prefetch_tensormap(&map_sl);
  }
  if (warp == 10 && lane == 0) {
    wgtc::prefetch_tensormap(&map_n);
    wgtc::prefetch_tensormap(&map_sn);
  }
  if (warp == 1) wgg::pair_tmem_alloc<CG>(tmem_slot, S::TMEM_COLS);
  wg_pdl_wait();
  wg_pdl_trigger();
  wgg::plan_groups(a.offsets, a.groups, a.rows, S::BN, start, tile0, atom0, a.dwords);
  wgtc::tc_fence_before();
  wgg::cluster_sync<S::CLUSTER>();
  wgtc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int64_t tiles = (int64_t)tile0[a.groups] * a.tiles_l;
  const int64_t t_first = blockIdx.x / S::CLUSTER, t_step = gridDim.x / S::CLUSTER;
  const uint32_t half = CG == 2 ? rank : 0;  // which lanes and columns of a pair's tile
  const int kt = a.out.alpha == 0.0f ? 0 : (a.k + BKE - 1) / BKE;
  auto gave_up = [&](unsigned bit) {
    atomicOr(a.dwords + WG_DW_ERROR, bit);
    *abort_flag = 1;
  };

  if (warp == 0 || warp == 10) {
    // ---- producers ----
    wgg::Ring<STAGES> ring;
    bool ok = true;
    const bool l_side = warp == 0;
    const uint32_t lead = wgg::leader_addr<CG>(full);
    for (int64_t t = t_first; t < tiles && ok; t += t_step) {
      const Tile x = tile_at<S>(a, t, start, tile0, atom0, kt, rank);
      const int cols = ((x.nv + S::NMMA_STEP - 1) & ~(S::NMMA_STEP - 1)) / CG;  // columns this CTA loads
      const int boxes = (cols + S::NBOX - 1) / S::NBOX;
      const int l0 = x.l0 + (int)half * BL, r0 = x.r0 + (int)half * cols;
      const int sl = x.g * a.l_atoms + l0 / 128;
      const uint32_t bytes = l_side ? (uint32_t)(S::L_BYTES + S::SF_L) : (uint32_t)(boxes * S::NBOX * 128 + S::SF_N);
      for (int kb = x.k_lo; kb < x.k_hi; kb++, ring.next()) {
        const int s = ring.s;
        ok = __all_sync(0xffffffffu, wgtc::mbar_wait_bounded(&empty[s], ring.round ^ 1u, WAIT_BUDGET));
        if (!ok) break;
        uint8_t *st = smem + (size_t)s * S::STAGE, *sf = st + S::L_BYTES + S::N_BYTES;
        const uint32_t at = lead + 8u * (uint32_t)s;
        if (wgg::elect()) {
          if (half == 0) wgtc::mbar_arrive_expect_tx(&full[s], CG * bytes);
          // (what lies past the last scale tile, or past the matrix's rows, arrives as zeros)
          if (l_side) {
            wgg::load_3d<CG>(st, &map_l, &full[s], at, kb * 128, l0, x.g);
            wgg::load_2d<CG>(sf, &map_sl, &full[s], at, kb * 256, sl);
          } else {
            for (int b = 0; b < boxes; b++)
              wgg::load_2d<CG>(st + S::L_BYTES + b * S::NBOX * 128, &map_n, &full[s], at, kb * 128, r0 + b * S::NBOX);
            wgg::load_2d<CG>(sf + S::SF_L, &map_sn, &full[s], at, kb * 256, x.n_atom);
          }
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) gave_up(WG_DERR_TMA_WAIT);
    // Let every copy (of both CTAs) land before the CTA can exit.
    for (int i = 0; i < STAGES && ok; i++, ring.next())
      if (!wgtc::mbar_wait_bounded(&empty[ring.s], ring.round ^ 1u, WAIT_BUDGET)) break;
  } else if (warp == 1) {
    if (half == 0) {
      // ---- MMA issuer ----
      wgg::Ring<STAGES> ring;
      int used = 0;
      uint32_t set = 0;  // which set of scale columns
      constexpr int segment = DRAIN ? DRAIN : 1 << 30;
      const uint32_t smem0 = wgtc::smem_addr(smem);
      const uint64_t desc_l0 = wgtc::smem_desc_kmajor(smem0, 128);
      const uint64_t desc_n0 = wgtc::smem_desc_kmajor(smem0 + S::L_BYTES, 128);
      const uint64_t desc_s0 = scales_desc(smem0 + S::L_BYTES + S::N_BYTES);
      bool ok = true;
      for (int64_t t = t_first; t < tiles && ok; t += t_step) {
        const Tile x = tile_at<S>(a, t, start, tile0, atom0, kt, rank);
        const int nmma = (x.nv + S::NMMA_STEP - 1) & ~(S::NMMA_STEP - 1);
        const uint32_t idesc0 = idesc_mxf4(S::TL, nmma, 0), idesc2 = idesc_mxf4(S::TL, nmma, 2);
        for (int kb0 = x.k_lo; kb0 < x.k_hi && ok; kb0 += segment, used++) {
          const int b = used % S::ACCS, kb1 = min(x.k_hi, kb0 + segment);
          const uint32_t d_tmem = tmem + (uint32_t)(b * S::BN);
          ok = __all_sync(0xffffffffu, wgg::leader_wait<CG>(&acc_empty[b], ((uint32_t)(used / S::ACCS) & 1u) ^ 1u));
          wgtc::tc_fence_after();
          for (int kb = kb0; kb < kb1 && ok; kb++, ring.next(), set ^= 1u) {
            ok = __all_sync(0xffffffffu, wgtc::mbar_wait_bounded(&full[ring.s], ring.round, WAIT_BUDGET));
            if (!ok) break;
            wgtc::tc_fence_after();
            const uint64_t at = (uint64_t)((uint32_t)ring.s * (S::STAGE >> 4));
            const uint64_t dl = desc_l0 + at, dn = desc_n0 + at, ds = desc_s0 + at;
            const uint32_t tl = tmem + S::SF_COL + set * S::SF_SET, tn = tl + 8;
            const int steps = (a.k - kb * BKE + 63) >> 6;
            if (wgg::elect()) {
#pragma unroll
              for (int j = 0; j < 2; j++) {
                copy_scales<CG>(tl + 4 * j, ds + 32 * j);
#pragma unroll
                for (int r = 0; r < S::NT; r++)
                  copy_scales<CG>(tn + 4 * S::NT * j + 4 * r, ds + 64 * (1 + r) + 32 * j);
              }
              if (steps >= 4) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                  mma_mxf4<CG>(d_tmem, dl + i * 2, dn + i * 2, i & 1 ? idesc2 : idesc0, tl + 4 * (i >> 1),
                               tn + 4 * S::NT * (i >> 1), i > 0 || kb > kb0 ? 1u : 0u);
              } else {
                for (int i = 0; i < steps; i++)
                  mma_mxf4<CG>(d_tmem, dl + i * 2, dn + i * 2, i & 1 ? idesc2 : idesc0, tl + 4 * (i >> 1),
                               tn + 4 * S::NT * (i >> 1), i > 0 || kb > kb0 ? 1u : 0u);
              }
              wgg::commit<CG>(&empty[ring.s]);
              if (kb == kb1 - 1) wgg::commit<CG>(&acc_full[b]);
            }
            __syncwarp();
          }
        }
      }
      if (!ok && lane == 0) gave_up(WG_DERR_MMA_WAIT);
    }
  } else if (warp >= 2 && warp < 2 + EPI_WARPS) {
    // ---- epilogue ----
    const int q = warp & 3, h = (warp - 2) >> 2;
    int used = 0;
    bool ok = true;
    for (int64_t t = t_first; t < tiles && ok; t += t_step) {
      const Tile x = tile_at<S>(a, t, start, tile0, atom0, kt, rank);
      const int valid = x.nv - h * S::CPT;  // columns this warp has (may be none)
      const int l = x.l0 + (int)half * BL + q * 32 + lane;
      const int64_t at = (int64_t)(x.r0 + h * S::CPT) * a.out.ldc + l;
      const uint32_t col = tmem + (uint32_t)(h * S::CPT) + ((uint32_t)(q * 32) << 16);
      float sum[S::CPT];
#pragma unroll
      for (int j = 0; j < S::CPT; j++) sum[j] = 0.0f;
      for (int kb0 = x.k_lo; kb0 < x.k_hi; kb0 += DRAIN ? DRAIN : 1 << 30, used++) {
        const int b = used % S::ACCS;
        ok = __all_sync(0xffffffffu, wgtc::mbar_wait_bounded(&acc_full[b], (uint32_t)(used / S::ACCS) & 1u, WAIT_BUDGET) &&
                                         *abort_flag == 0);
        if (!ok) {
          if (lane == 0) gave_up(WG_DERR_MMA_WAIT);
          break;
        }
        wgtc::tc_fence_after();
        wgg::drain<S::CPT>(col + (uint32_t)(b * S::BN), valid, kb0 == x.k_lo, sum);
        wgtc::tc_fence_before();
        __syncwarp();
        if (lane == 0) wgg::leader_arrive<CG>(&acc_empty[b]);
      }
      if (!ok) break;
      bool mine = true;
      if constexpr (S::P > 1) {
        if (kt) mine = wgg::join_parts<S::P, S::BN, S::CPT>(parts, rank, h * S::CPT, q * 32 + lane, valid, x.nv,
                                                              warp == 2, t + t_step < tiles, sum, &ok);
        else mine = rank == 0;
        if (!ok) {
          if (lane == 0) gave_up(WG_DERR_MMA_WAIT);
          break;
        }
      }
      if (mine) wgg::store_sums<S::CPT, DRAIN == SEG && S::P == 1>(a.out, at, l < a.n, valid, sum);
    }
  }

  wgtc::tc_fence_before();
  __syncwarp();
  wgg::cluster_sync<S::CLUSTER>();
  if (warp == 1) {
    wgtc::tc_fence_after();
    wgg::pair_tmem_dealloc<CG>(tmem, S::TMEM_COLS);
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
  return groups > 0 ? wgg::check_offsets(offsets) : WG_OK;
}

wg_status launch_quant(wg_device *d, const char *family, void (*kern)(const QuantArgs), const QuantArgs &a, int64_t ctas) {
  if (ctas >= LIM) return wg_fail(WG_ERR_INVALID_ARGUMENT, "too many elements for one call");
  wg_launch_scope scope(d, family);
  WG_CUDA(wg_launch_pdl(kern, dim3((unsigned)ctas), dim3(256), 0, d->stream, a));
  WG_CUDA(cudaGetLastError());
  return WG_OK;
}
int64_t row_tiles(const QuantArgs &a) { return a.offsets ? tiles_of(a.rows) + a.groups : (int64_t)a.batch * a.tiles_r; }

// The row forms: CTAs of quarters of a tile pair, of whole ones for 16-bit matrices
// of whole 16-byte units with at least three pairs an SM. us, whole against quarters,
// bf16: 1000 x 1024 4.3 / 2.4 (back 4.4 / 2.4), 2048 x 4096 7.6 / 7.1, 4096 x 4096
// 10.1 / 11.3 (back 9.1 / 10.3), 8192 x 8192 32.0 / 37.8 (back 33.1 / 39.3), unaligned 4000 x 4001 20.5 /
// 17.4; fp32: 4096 x 4096 14.1 / 13.9, 8192 x 8192 47.2 / 45.6 (back 55.7 / 49.8).
template <class T>
wg_status launch_rows(wg_device *d, const char *family, bool back, const QuantArgs &a) {
  const int64_t pairs = row_tiles(a) * ((a.tiles_c + 1) / 2);
  const bool aligned = (((uintptr_t)a.X | (uintptr_t)a.ldx * sizeof(T) |
                         (a.batch > 1 ? (uintptr_t)a.strideX * sizeof(T) : 0)) & 15) == 0;
  if constexpr (sizeof(T) == 2)
    if (aligned && pairs >= (int64_t)3 * d->sm_count)
      return launch_quant(d, family, back ? mx_dequantize<T, 8> : mx_quantize<T, 8>, a, pairs);
  return launch_quant(d, family, !back     ? mx_quantize<T, 32>
                                 : aligned ? mx_dequantize<T, 32>
                                           : mx_dequantize_unaligned<T>, a, pairs * 4);
}
wg_status launch_rows_of(wg_device *d, const char *family, bool back, const QuantArgs &a) {
  return a.xtype == WG_TYPE_F32    ? launch_rows<float>(d, family, back, a)
         : a.xtype == WG_TYPE_BF16 ? launch_rows<__nv_bfloat16>(d, family, back, a)
                                   : launch_rows<__half>(d, family, back, a);
}

bool encode(CUtensorMap *map, CUtensorMapDataType type, const void *ptr, int rank, const cuuint64_t *dims,
            const cuuint64_t *strides, const cuuint32_t *box, CUtensorMapSwizzle swizzle) {
  wg_encode_tiled_fn fn = wg_encode_tiled();
  if (!fn) return false;
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, type, rank, const_cast<void *>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Operands {
  const uint8_t *A, *As, *B, *Bs;
};

template <class S, int DRAIN>
wg_status launch_as(wg_device *d, const char *family, Args &a, const CUtensorMap (&m)[4]) {
  const int64_t most = ((int64_t)a.rows / S::BN + a.groups) * a.tiles_l;
  const unsigned grid = S::CLUSTER * (unsigned)std::max<int64_t>(1, std::min<int64_t>(most, d->sm_count / S::CLUSTER));
  wg_launch_scope scope(d, family);
  WG_CUDA(wg_kernel_smem(mx_gemm_kernel<S, DRAIN>, SMEM_LIMIT));
  WG_CUDA((wgg::launch<S::CLUSTER>(mx_gemm_kernel<S, DRAIN>, grid, 352, S::smem(a.groups), d->stream, m[0], m[1], m[2], m[3], a)));
  WG_CUDA(cudaGetLastError());
  return WG_OK;
}

template <class S>
wg_status launch_gemm(wg_device *d, const char *family, Args &a, const Operands &o) {
  CUtensorMap m[4];
  memset(m, 0, sizeof m);
  a.tiles_l = (a.n + S::TL - 1) / S::TL;
  if (a.out.alpha != 0.0f) {
    const cuuint64_t pitch = (cuuint64_t)pitch_of(a.k), words = (cuuint64_t)tiles_of(a.k) * 128;
    const cuuint64_t dl[3] = {pitch, (cuuint64_t)a.n, (cuuint64_t)a.groups}, sl[2] = {pitch, pitch * (cuuint64_t)a.n};
    const cuuint32_t bl[3] = {128, (cuuint32_t)BL, 1};
    const cuuint64_t dn[2] = {pitch, (cuuint64_t)a.rows};
    const cuuint32_t bn[2] = {128, (cuuint32_t)S::NBOX};
    // Scales: rows of tiles, as 32-bit words; a box is two tiles long.
    const cuuint64_t ss = words * 4;
    const cuuint64_t dsl[2] = {words, (cuuint64_t)a.l_atoms * (cuuint64_t)a.groups};
    const cuuint64_t dsn[2] = {words, (cuuint64_t)tiles_of(a.rows) + (a.offsets ? (cuuint64_t)a.groups : 0)};
    const cuuint32_t bsl[2] = {256, 1}, bsn[2] = {256, (cuuint32_t)S::NT};
    const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8, u32 = CU_TENSOR_MAP_DATA_TYPE_UINT32;
    const CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_128B, no = CU_TENSOR_MAP_SWIZZLE_NONE;
    if (!encode(&m[0], u8, o.B, 3, dl, sl, bl, sw) || !encode(&m[1], u8, o.A, 2, dn, sl, bn, sw) ||
        !encode(&m[2], u32, o.Bs, 2, dsl, &ss, bsl, no) || !encode(&m[3], u32, o.As, 2, dsn, &ss, bsn, no))
      return wg_fail(WG_ERR_INVALID_ARGUMENT, "the operands' sizes exceed what a tensor map describes");
  }
  if constexpr (S::P > 1) {
    return launch_as<S, SEG>(d, family, a, m);
  } else {
    if (a.out.type == WG_TYPE_F32) return a.k > SEG * BKE ? launch_as<S, SEG>(d, family, a, m) : launch_as<S, 0>(d, family, a, m);
    return a.k > whole_rows(a.out.type) ? launch_as<S, LONG>(d, family, a, m) : launch_as<S, 0>(d, family, a, m);
  }
}

// The form with the least modelled time, as for the 16-bit products (grouped.cu);
// joining parts costs about 2700 clocks, a pair's start and single accumulator
// 3500. us in a CUDA graph, operands in L2, m x n x k (groups), the chosen form's starred:
//                            pair  128 columns  32 columns  ... split 2  split 4
//   1024 x 4096 x 4096 (1)   12.0*    12.8         -            -         -
//   128 x 8192 x 4096 (1)     9.8      8.1*        -            -         -
//   1500 x 2048 x 4096 (32)  30.9     29.8*        -            -         -
//   16 x 8192 x 4096 (1)      7.3      6.6        6.2*         6.4      11.0
//   16 x 2048 x 8192 (1)     10.6      9.4        9.2          7.2       6.0*
//   30 x 2048 x 2048 (16)     9.9      9.2        7.9*         9.8      24.2
// (a split of 128-column tiles won nowhere by more than 4 % and is not built).
// A 32-column form needs every group to fit it, which only the number of all rows can show here.
enum Form { PAIR_256, ONE_128, ONE_32, SPLIT_32_2, SPLIT_32_4, FORMS };
Form choose(const wg_device *d, const Args &a) {
  static const struct { int cg, bn, p; } forms[FORMS] = {{2, 256, 1}, {1, 128, 1}, {1, 32, 1}, {1, 32, 2}, {1, 32, 4}};
  const int64_t groups = std::max<int64_t>(1, std::min(a.groups, a.rows));
  const int64_t cols = (a.rows + groups - 1) / groups, kt = std::max<int64_t>(1, (a.k + BKE - 1) / BKE);
  Form best = ONE_128;
  double least = 1e300;
  for (int i = 0; i < FORMS; i++) {
    const auto f = forms[i];
    if (f.bn == 32 && a.rows > 32) continue;
    const int64_t nt = (cols + f.bn - 1) / f.bn, nv = (cols + nt - 1) / nt;
    const int64_t tl = (a.n + f.cg * BL - 1) / (f.cg * BL);
    const int64_t slots = f.p == 4 ? d->sm_count * 3 / 16 : d->sm_count / (f.cg * f.p);
    const int64_t rounds = (tl * groups * nt + slots - 1) / slots;
    const int64_t box = std::min<int64_t>(f.bn, 64), lines = (nv / f.cg + box - 1) / box * box;
    const double block = std::max({nv * 2.0, ((BL + lines) * 128 + 2048) / 65.0, 300.0});
    const double tail = (double)BL * nv * (a.out.type == WG_TYPE_F32 ? 4 : 2) / 20 +
                        (f.p > 1 ? 2700 : f.cg > 1 ? 3500 : 0);
    const double t = rounds * (double)((kt + f.p - 1) / f.p) * block + tail;
    if (t < least) {
      least = t;
      best = (Form)i;
    }
  }
  return best;
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
  if ((st = wgg::check_aligned("C", C, ctype)) != WG_OK || (st = wgg::check_offsets(offsets)) != WG_OK) return st;
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
  a.l_atoms = (int)tiles_of(n);
  a.offsets = offsets;
  a.out = {C, ldc, alpha, beta, ctype};
  a.dwords = d->dwords;
  const Operands o = {static_cast<const uint8_t *>(A), static_cast<const uint8_t *>(As),
                      static_cast<const uint8_t *>(B), static_cast<const uint8_t *>(Bs)};
  return wg_timed(d, gpu_ms, [&] {
    const Form form = choose(d, a);
    switch (form) {
      case PAIR_256: return launch_gemm<Shape<2, 256>>(d, family, a, o);
      case ONE_128: return launch_gemm<Shape<1, 128>>(d, family, a, o);
      case ONE_32: return launch_gemm<Shape<1, 32>>(d, family, a, o);
      case SPLIT_32_2: return launch_gemm<Shape<1, 32, 2>>(d, family, a, o);
      default: return launch_gemm<Shape<1, 32, 4>>(d, family, a, o);
    }
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
  if ((st = wgg::check_aligned("X", X, type)) != WG_OK || (st = check_matrix("out", codes, scales)) != WG_OK ||
      (st = wgg::check_arch(d)) != WG_OK)
    return st;
  if (batch >= LIM || batch * tiles_of(rows) >= LIM) return wg_fail(WG_ERR_INVALID_ARGUMENT, "too many elements for one call");
  wg_device_guard guard(d->ordinal);
  QuantArgs a = {X, ldx, strideX, type, (int)rows, (int)cols, static_cast<uint8_t *>(codes),
                 static_cast<uint8_t *>(scales), pitch_of(cols), (int)tiles_of(rows), (int)tiles_of(cols), (int)batch,
                 groups ? offsets : nullptr, (int)groups, d->dwords};
  return wg_timed(d, gpu_ms, [&] {
    if (!trans) return launch_rows_of(d, "mx_quantize", false, a);
    return launch_quant(d, "mx_quantize", type == WG_TYPE_F32    ? mx_quantize_t<float>
                                          : type == WG_TYPE_BF16 ? mx_quantize_t<__nv_bfloat16>
                                                                 : mx_quantize_t<__half>, a, row_tiles(a) * a.tiles_c);
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
  if (batch > 1 && !wgg::apart(strideX, rows, cols, ldx))
    return wg_fail(WG_ERR_INVALID_ARGUMENT, "strideX must be at least one matrix of X.");
  if (batch == 0 || rows == 0 || cols == 0) return WG_OK;
  if (!X) return wg_fail(WG_ERR_INVALID_ARGUMENT, "operand pointer is NULL");
  if ((st = wgg::check_aligned("X", X, type)) != WG_OK || (st = check_matrix("x", codes, scales)) != WG_OK ||
      (st = wgg::check_arch(d)) != WG_OK)
    return st;
  if (batch >= LIM || batch * tiles_of(rows) >= LIM) return wg_fail(WG_ERR_INVALID_ARGUMENT, "too many elements for one call");
  wg_device_guard guard(d->ordinal);
  QuantArgs a = {X, ldx, strideX, type, (int)rows, (int)cols, static_cast<uint8_t *>(const_cast<void *>(codes)),
                 static_cast<uint8_t *>(const_cast<void *>(scales)), pitch_of(cols), (int)tiles_of(rows),
                 (int)tiles_of(cols), (int)batch, groups ? offsets : nullptr, (int)groups, d->dwords};
  return wg_timed(d, gpu_ms, [&] { return launch_rows_of(d, "mx_dequantize", true, a); });
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
