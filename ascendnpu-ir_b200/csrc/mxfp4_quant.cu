// mxfp4_quant.cu -- quantisation to and from microscaled 4-bit floats (the OCP MX format MXFP4): 32 consecutive
// elements along the contracted axis share one exponent byte (E8M0: 2^(byte - 127), 255 = NaN), an element is e2m1
// (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte with the even element in the lower half.
//
//   byte = clamp(floor(log2(max |x|)) - 2 + 127, 0, ..),   code = rne_e2m1(x * 2^(127 - byte)), stopped at +-6
//
// A power of two divides exactly, so every rounding but the element's own is avoided and the result does not depend on
// how the work is cut: the exponent is read off the bits of the largest magnitude (its exponent field less 2), and
// x * 2^(127 - byte) is exact wherever it could matter (only what rounds to zero anyway can fall under the normals).
// A block that holds a NaN or an infinity gets the exponent byte 255 and codes 0.  Missing elements of a last block
// are zeros, the unused half of a row's last byte is 0.
//
// Both directions of a matrix can come out of one read: blocks along the rows (what C = A * B^T contracts) and blocks
// down the columns with the result transposed (what the products of a backward pass contract).
#include "tc_ptx.cuh"

namespace bsir {
namespace {

constexpr int kBlock = 32;

// index -> row without a division instruction: row = (i * magic) >> shift for i < 2^31 (round-up method; the divisor
// of a vector index is the number of vectors in a padded row)
struct FastDiv {
  uint32_t d, magic, shift;
};
FastDiv make_fastdiv(uint32_t d) {
  FastDiv f{d, 0, 0};
  while ((1ull << f.shift) < d) ++f.shift;
  f.magic = static_cast<uint32_t>(((1ull << 32) * ((1ull << f.shift) - d)) / d + 1);
  return f;
}
__device__ __forceinline__ uint32_t fast_div(const FastDiv &f, uint32_t i) {
  return (__umulhi(i, f.magic) + i) >> f.shift;   // i < 2^31 and the high product < i: the sum cannot wrap
}

// the largest magnitude's bits (NaN > infinity > numbers) -> exponent byte
__device__ __forceinline__ uint32_t scale_byte(uint32_t abs_bits) {
  const uint32_t e = abs_bits >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// 2^(127 - byte) as float; byte <= 252 unless 255
__device__ __forceinline__ float inv_scale(uint32_t byte) { return __uint_as_float((254u - (byte > 252u ? 252u : byte)) << 23); }

// eight values -> eight codes, element 0 in the lowest half byte.  The conversion rounds to nearest even, stops at
// +-6 and keeps the sign of what rounds to zero.
__device__ __forceinline__ uint32_t pack_e2m1x8(const float *v) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// eight codes -> eight values (exact in f16, hence in f32)
__device__ __forceinline__ void unpack_e2m1x8(uint32_t q, float *v) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(q));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = f16lo_to_f32(h[i]);
    v[2 * i + 1] = f16hi_to_f32(h[i]);
  }
}

// Two 16-bit floats at once: the larger magnitude with some sign (a NaN stays one), one instruction where clearing the
// signs and comparing bits is two.  A bf16 times a power of two is exact, so pairs are scaled before they are widened (the power and its product
// with anything that does not round to zero are bf16 numbers; f16's exponent range is too short for that).
template <int DT> __device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (DT == BSIR_BF16) asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// magnitude bits of a 16-bit float as those of the f32 of the same value (NaN and infinity stay what they are)
template <int DT> __device__ __forceinline__ uint32_t widen_abs(uint32_t h) {
  if constexpr (DT == BSIR_BF16) return h << 16;
  else return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(h))));
}
// eight elements as they lie in memory -> codes and the block's exponent byte, by the four lanes that hold the block
template <int DT>
__device__ __forceinline__ uint32_t quant8(const uint32_t *w, uint32_t *byte_out) {
  constexpr int kPer = FloatTraits<DT>::kPerWord;
  uint32_t m;
  if constexpr (DT == BSIR_F32) {
    m = w[0] & 0x7fffffffu;
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max(m, w[i] & 0x7fffffffu);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  } else {
    uint32_t h = max_abs2<DT>(max_abs2<DT>(w[0], w[1]), max_abs2<DT>(w[2], w[3]));
    h = max_abs2<DT>(h, __shfl_xor_sync(0xffffffffu, h, 1));
    h = max_abs2<DT>(h, __shfl_xor_sync(0xffffffffu, h, 2));
    m = widen_abs<DT>(max(h & 0x7fffu, h >> 16 & 0x7fffu));
  }
  const uint32_t byte = scale_byte(m);
  const float inv = inv_scale(byte);
  float v[8];
  if constexpr (DT == BSIR_BF16) {
    const uint32_t inv2 = __float_as_uint(inv) | (__float_as_uint(inv) >> 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) FloatTraits<DT>::unpack(mul_bf16x2(w[i], inv2), v + 2 * i);
  } else {
#pragma unroll
    for (int i = 0; i < 8 / kPer; ++i) FloatTraits<DT>::unpack(w[i], v + i * kPer);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], inv);
  }
  *byte_out = byte;
  return byte == 255u ? 0u : pack_e2m1x8(v);
}

template <int DT> __device__ __forceinline__ float load_elem(const void *x, int64_t i) {
  if constexpr (DT == BSIR_F32) return static_cast<const float *>(x)[i];
  else if constexpr (DT == BSIR_F16) return __half2float(__ushort_as_half(static_cast<const unsigned short *>(x)[i]));
  else return __uint_as_float(static_cast<uint32_t>(static_cast<const unsigned short *>(x)[i]) << 16);
}

// eight consecutive elements of a row as they lie in memory; those at or behind `cols` are zeros
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const void *x, int64_t row_at, int64_t c, int64_t cols, uint32_t *w) {
  constexpr int kPer = FloatTraits<DT>::kPerWord, kWords = 8 / kPer;
  if constexpr (VEC) {                 // cols % 8 == 0: a vector is all inside or all outside
    if (c < cols) {
      const char *src = static_cast<const char *>(x) + (row_at + c) * (4 / kPer);
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const Vec16 b = ld_stream(src + 4 * i);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[i + k] = b.w[k];
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? load_elem<DT>(x, row_at + c + i) : 0.0f;
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = FloatTraits<DT>::pack(v + i * kPer);
  }
}

struct QuantParams {
  int64_t rows, cols;
  const void *x;
  int64_t xs;                 // row stride of x, elements
  uint8_t *q;                 // blocks along the rows, may be null
  int64_t qs;
  uint8_t *s;
  int64_t ss;
  uint8_t *qt;                // blocks down the columns, transposed, may be null
  int64_t qts;
  uint8_t *st;
  int64_t sts;
  FastDiv div;
  uint32_t nvec;              // vectors of eight in all rows, rows padded to whole blocks
  int q_words, qt_words;      // 4-byte / 16-byte stores of codes are aligned
};

__device__ __forceinline__ void store_codes(uint8_t *dst, uint32_t codes, int nbytes, bool words) {
  if (words && nbytes >= 4) {
    *reinterpret_cast<uint32_t *>(dst) = codes;
  } else {
    for (int i = 0; i < 4 && i < nbytes; ++i) dst[i] = static_cast<uint8_t>(codes >> (8 * i));
  }
}

// Blocks along the rows: a lane takes eight elements (16 bytes of a 16-bit type), four lanes are a block and meet in
// two shuffles; a warp's codes leave as 128 consecutive bytes.  Four vectors a thread are loaded before the first is
// used.  FLAT: rows of whole blocks that follow one another without gaps in x, codes and exponents, so that a vector's
// number is all the addressing it takes.
constexpr int kRowVecs = 4;
template <int DT, bool VEC, bool FLAT>
__global__ void __launch_bounds__(256) mxfp4_rows_kernel(QuantParams p) {
  constexpr int kWords = 8 / FloatTraits<DT>::kPerWord;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t v0 = blockIdx.x * (256u * kRowVecs) + threadIdx.x;
  uint32_t w[kRowVecs][kWords];
  if constexpr (FLAT) {
    const char *src = static_cast<const char *>(p.x) + static_cast<uint64_t>(v0) * (4 * kWords);
#pragma unroll
    for (int u = 0; u < kRowVecs; ++u) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[u][i] = 0u;
      if (v0 + u * 256u < p.nvec) {
#pragma unroll
        for (int i = 0; i < kWords; i += 4) {
          const Vec16 b = ld_stream(src + u * 256 * 4 * kWords + 4 * i);
#pragma unroll
          for (int k = 0; k < 4; ++k) w[u][i + k] = b.w[k];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kRowVecs; ++u) {
      uint32_t byte;
      const uint32_t codes = quant8<DT>(w[u], &byte);
      const uint32_t i = v0 + u * 256u;
      if (i < p.nvec) {
        reinterpret_cast<uint32_t *>(p.q)[i] = codes;
        if ((threadIdx.x & 3) == 0) p.s[i >> 2] = static_cast<uint8_t>(byte);
      }
    }
  } else {
    uint32_t row[kRowVecs], col[kRowVecs];
#pragma unroll
    for (int u = 0; u < kRowVecs; ++u) {
      const uint32_t i = v0 + u * 256u;
      row[u] = fast_div(p.div, i);
      col[u] = (i - row[u] * p.div.d) * 8u;
      load8<DT, VEC>(p.x, static_cast<int64_t>(row[u]) * p.xs, col[u], i < p.nvec ? p.cols : 0, w[u]);
    }
#pragma unroll
    for (int u = 0; u < kRowVecs; ++u) {
      uint32_t byte;
      const uint32_t codes = quant8<DT>(w[u], &byte);
      if (v0 + u * 256u < p.nvec && col[u] < p.cols) {
        const int nbytes = static_cast<int>(min(static_cast<int64_t>(4), (p.cols - col[u] + 1) / 2));
        store_codes(p.q + static_cast<int64_t>(row[u]) * p.qs + col[u] / 2, codes, nbytes, p.q_words);
        if ((threadIdx.x & 3) == 0) p.s[static_cast<int64_t>(row[u]) * p.ss + col[u] / kBlock] = static_cast<uint8_t>(byte);
      }
    }
  }
}

// Blocks down the columns, and along the rows as well when `q` is wanted, on tiles of kTR rows x 64 columns in shared
// memory (128 bytes of a row of a 16-bit type).  Down the columns a thread takes two neighbouring columns of a 32-row block -- a warp reads one row of the tile at a time -- and its two blocks'
// codes (16 bytes each) go through shared memory so that a column's codes leave as kTR / 2 consecutive bytes.
constexpr int kTC = 64;
constexpr int kTR = 128;
constexpr int kColThreads = 128;
constexpr int kCodeRow = kTR / 2 + 16;                   // bytes of a column's codes, padded against bank conflicts
constexpr int kColPieces = kTR / kBlock;                 // 16-byte pieces (blocks) of a column of a tile

// half of a swizzled row of a tile of 16-bit floats (`row8`: the row modulo 8): one block along the row
template <int DT>
__device__ __forceinline__ uint4 quant_block(const uint8_t *row, int half, int row8, uint32_t *byte_out) {
  uint32_t w[16];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 v = *reinterpret_cast<const uint4 *>(row + (((4 * half + j) ^ row8) * 16));
    w[4 * j] = v.x; w[4 * j + 1] = v.y; w[4 * j + 2] = v.z; w[4 * j + 3] = v.w;
  }
  uint32_t h = w[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) h = max_abs2<DT>(h, w[i]);
  const uint32_t byte = scale_byte(widen_abs<DT>(max(h & 0x7fffu, h >> 16 & 0x7fffu)));
  const float inv = inv_scale(byte);
  const uint32_t inv2 = __float_as_uint(inv) | (__float_as_uint(inv) >> 16);
  uint32_t q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == BSIR_BF16) {
        FloatTraits<DT>::unpack(mul_bf16x2(w[4 * j + i], inv2), v + 2 * i);
      } else {
        FloatTraits<DT>::unpack(w[4 * j + i], v + 2 * i);
        v[2 * i] = __fmul_rn(v[2 * i], inv);
        v[2 * i + 1] = __fmul_rn(v[2 * i + 1], inv);
      }
    }
    q[j] = pack_e2m1x8(v);
  }
  *byte_out = byte;
  return byte == 255u ? make_uint4(0, 0, 0, 0) : make_uint4(q[0], q[1], q[2], q[3]);
}

// this warp's 32-row block b of the tile, lane = a pair of columns -> codes and exponents down the columns
// (SWZ: 16-byte pieces of a row of the tile permuted by the row, as the copy engine's 128-byte swizzle leaves them)
template <int DT, bool SWZ = false>
__device__ __forceinline__ void quant_down(const uint8_t *tile, uint8_t *codes_s, uint8_t (*scale_s)[kColPieces], int b) {
  constexpr int EB = 4 / FloatTraits<DT>::kPerWord;
  const int lane = threadIdx.x & 31;
  uint32_t byte[2];
  uint32_t q0[4], q1[4];
  const uint8_t *src = tile + (b * kBlock * kTC + 2 * lane) * EB;
  if constexpr (DT == BSIR_F32) {
    uint32_t m0 = 0, m1 = 0;
    float2 x[kBlock];
#pragma unroll
    for (int r = 0; r < kBlock; ++r) {
      x[r] = *reinterpret_cast<const float2 *>(src + r * kTC * EB);
      m0 = max(m0, __float_as_uint(x[r].x) & 0x7fffffffu);
      m1 = max(m1, __float_as_uint(x[r].y) & 0x7fffffffu);
    }
    byte[0] = scale_byte(m0);
    byte[1] = scale_byte(m1);
    const float i0 = inv_scale(byte[0]), i1 = inv_scale(byte[1]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float v[8], y[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        v[r] = __fmul_rn(x[8 * j + r].x, i0);
        y[r] = __fmul_rn(x[8 * j + r].y, i1);
      }
      q0[j] = pack_e2m1x8(v);
      q1[j] = pack_e2m1x8(y);
    }
  } else {
    uint32_t x[kBlock], m = 0;
#pragma unroll
    for (int r = 0; r < kBlock; ++r) {
      x[r] = *reinterpret_cast<const uint32_t *>(SWZ ? tile + (b * kBlock + r) * kTC * EB + ((4 * lane) ^ ((r & 7) * 16)) : src + r * kTC * EB);
      m = max_abs2<DT>(m, x[r]);
    }
    byte[0] = scale_byte(widen_abs<DT>(m & 0x7fffu));
    byte[1] = scale_byte(widen_abs<DT>(m >> 16 & 0x7fffu));
    const float i0 = inv_scale(byte[0]), i1 = inv_scale(byte[1]);
    const uint32_t inv2 = (__float_as_uint(i0) >> 16) | __float_as_uint(i1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float v[8], y[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        float f[2];
        if constexpr (DT == BSIR_BF16) {
          FloatTraits<DT>::unpack(mul_bf16x2(x[8 * j + r], inv2), f);
        } else {
          FloatTraits<DT>::unpack(x[8 * j + r], f);
          f[0] = __fmul_rn(f[0], i0);
          f[1] = __fmul_rn(f[1], i1);
        }
        v[r] = f[0];
        y[r] = f[1];
      }
      q0[j] = pack_e2m1x8(v);
      q1[j] = pack_e2m1x8(y);
    }
  }
  *reinterpret_cast<uint4 *>(codes_s + 2 * lane * kCodeRow + b * 16) = byte[0] == 255u ? make_uint4(0, 0, 0, 0) : make_uint4(q0[0], q0[1], q0[2], q0[3]);
  *reinterpret_cast<uint4 *>(codes_s + (2 * lane + 1) * kCodeRow + b * 16) = byte[1] == 255u ? make_uint4(0, 0, 0, 0) : make_uint4(q1[0], q1[1], q1[2], q1[3]);
  scale_s[2 * lane][b] = static_cast<uint8_t>(byte[0]);
  scale_s[2 * lane + 1][b] = static_cast<uint8_t>(byte[1]);
}
// the tile's codes and exponents down the columns, from shared memory to their rows
__device__ __forceinline__ void store_down(const QuantParams &p, const uint8_t *codes_s, const uint8_t (*scale_s)[kColPieces], int64_t r0, int64_t c0) {
  const int64_t code_bytes = (p.rows + 1) / 2, blocks = (p.rows + kBlock - 1) / kBlock;
  for (int i = threadIdx.x; i < kTC * kColPieces; i += kColThreads) {
    const int c = i / kColPieces, b = i % kColPieces;
    const int64_t col = c0 + c, at = r0 / 2 + b * 16;
    if (col >= p.cols || at >= code_bytes) continue;
    uint8_t *dst = p.qt + col * p.qts + at;
    const uint8_t *src = codes_s + c * kCodeRow + b * 16;
    if (p.qt_words && at + 16 <= code_bytes) {
      *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(src);
    } else {
      for (int j = 0; j < 16 && at + j < code_bytes; ++j) dst[j] = src[j];
    }
    if (r0 / kBlock + b < blocks) p.st[col * p.sts + r0 / kBlock + b] = scale_s[c][b];
  }
}

// Tiles by the copy engine, two a CTA, the next one on its way while this one is worked on (a CTA that loads its tile
// itself, works and stores, and is then replaced, reached 0.76 of the copy rate on bf16 and 0.70 on f32 down the columns;
// this 0.85 and 0.93).  Rows and columns behind the ends arrive as zeros.  One barrier a tile: the codes' staging is used
// in turns as well.  BOTH: four more warps make the blocks along the rows of the same tile.  Instructions bound that
// (eight elements a lane and two shuffles a block, as in the kernel above: 55 us on bf16 [16384, 4096]), so on 16-bit types
// a thread takes a whole block, 64 bytes of a row, which the 128-byte swizzle spreads over the banks: 40.5 us, 0.78 of the
// copy rate; f32, with eight elements a lane, 64.5, 0.80.
template <int DT, bool BOTH>
__global__ void __launch_bounds__(BOTH ? 2 * kColThreads : kColThreads, BOTH ? (DT == BSIR_F32 ? 3 : 4) : 1)
    mxfp4_cols_tma_kernel(const __grid_constant__ CUtensorMap tmap, QuantParams p, int64_t tiles, int64_t col_tiles, int *err) {
  constexpr int EB = 4 / FloatTraits<DT>::kPerWord, kWords = 8 / FloatTraits<DT>::kPerWord, kTile = kTR * kTC * EB;
  extern __shared__ uint8_t raw[];
  __shared__ uint8_t scale_s[2][kTC][kColPieces];
  __shared__ uint64_t full_s[2];
  __shared__ int abort_s;
  constexpr bool kSwz = BOTH && DT != BSIR_F32;
  constexpr uint32_t kAlign = kSwz ? 1024 : 128;
  const uint32_t base = (smem_u32(raw) + kAlign - 1) & ~(kAlign - 1);
  uint8_t *tile_s = raw + (base - smem_u32(raw));
  uint8_t *codes_s = tile_s + 2 * kTile;
  const bool q_vec = BOTH && ((reinterpret_cast<uintptr_t>(p.q) | static_cast<uintptr_t>(p.qs)) & 15) == 0;
  const int tid = threadIdx.x;
  auto load = [&](int64_t t, int b) {          // by thread 0
    const int64_t row_tile = t / col_tiles;
    mbar_expect_tx(smem_u32(&full_s[b]), kTile);
    tma_load_2d(base + b * kTile, &tmap, static_cast<int>((t - row_tile * col_tiles) * kTC * EB), static_cast<int>(row_tile * kTR), smem_u32(&full_s[b]));
  };
  if (tid == 0) {
    mbar_init(smem_u32(&full_s[0]), 1);
    mbar_init(smem_u32(&full_s[1]), 1);
    abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tmap(&tmap);
  }
  pdl_launch_dependents();
  pdl_wait();
  __syncthreads();
  if (tid == 0) {
    load(blockIdx.x, 0);
    if (blockIdx.x + gridDim.x < tiles) load(blockIdx.x + gridDim.x, 1);
  }
  int n = 0;
  int64_t t = blockIdx.x;
  for (; t < tiles; t += gridDim.x, ++n) {
    const int b = n & 1;
    const bool ok = mbar_wait(smem_u32(&full_s[b]), (n >> 1) & 1, &abort_s, err);
    const int64_t row_tile = t / col_tiles, r0 = row_tile * kTR, c0 = (t - row_tile * col_tiles) * kTC;
    const uint8_t *tile = tile_s + b * kTile;
    uint8_t *codes = codes_s + b * (kTC * kCodeRow);
    if (!BOTH || tid < kColThreads) {
      quant_down<DT, kSwz>(tile, codes, scale_s[b], tid >> 5);
    } else if constexpr (kSwz) {
      // a block a thread, two of them: nothing to pass between lanes, and one exponent's arithmetic for 32 elements
      const int rows = static_cast<int>(min(static_cast<int64_t>(kTR), p.rows - r0));       // of the tile
      const int half = tid & 1;
      const int64_t col = c0 + half * kBlock, left = (p.cols - col + 1) / 2;
      const int nbytes = left < 0 ? 0 : left < 16 ? static_cast<int>(left) : 16;
#pragma unroll 1
      for (int row = (tid - kColThreads) >> 1; row < kTR; row += kColThreads / 2) {
        uint32_t byte;
        const uint4 q16 = quant_block<DT>(tile + row * kTC * EB, half, row & 7, &byte);
        if (row >= rows || nbytes <= 0) continue;
        uint8_t *q = p.q + (r0 + row) * p.qs + col / 2;
        if (q_vec && nbytes == 16) {
          *reinterpret_cast<uint4 *>(q) = q16;
        } else {
          const uint32_t w[4] = {q16.x, q16.y, q16.z, q16.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) store_codes(q + 4 * j, w[j], nbytes - 4 * j, p.q_words);
        }
        p.s[(r0 + row) * p.ss + col / kBlock] = static_cast<uint8_t>(byte);
      }
    } else {
      const int r = (tid - kColThreads) >> 3, c = (tid & 7) * 8;
      const int rows = static_cast<int>(min(static_cast<int64_t>(kTR), p.rows - r0));       // of the tile
      const int nbytes = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(4), (p.cols - c0 - c + 1) / 2)));
      uint8_t *q = p.q + (r0 + r) * p.qs + (c0 + c) / 2, *s = p.s + (r0 + r) * p.ss + (c0 + c) / kBlock;
      const bool whole = rows == kTR && c0 + kTC <= p.cols && p.q_words;
#pragma unroll
      for (int u = 0; u < kTR * 8 / kColThreads; ++u) {
        const int row = r + u * (kColThreads / 8);
        uint32_t w[kWords], byte;
#pragma unroll
        for (int j = 0; j < kWords; j += 4) {
          const uint4 v = *reinterpret_cast<const uint4 *>(tile + (row * kTC + c) * EB + 4 * j);
          w[j] = v.x; w[j + 1] = v.y; w[j + 2] = v.z; w[j + 3] = v.w;
        }
        const uint32_t q8 = quant8<DT>(w, &byte);
        if (whole) {
          *reinterpret_cast<uint32_t *>(q) = q8;
          if ((tid & 3) == 0) *s = static_cast<uint8_t>(byte);
        } else if (row < rows && nbytes > 0) {
          store_codes(q, q8, nbytes, p.q_words);
          if ((tid & 3) == 0) *s = static_cast<uint8_t>(byte);
        }
        q += (kColThreads / 8) * p.qs;
        s += (kColThreads / 8) * p.ss;
      }
    }
    if (!__syncthreads_and(ok)) break;
    if (tid == 0 && t + 2 * static_cast<int64_t>(gridDim.x) < tiles) load(t + 2 * static_cast<int64_t>(gridDim.x), b);
    if (!BOTH || tid < kColThreads) store_down(p, codes, scale_s[b], r0, c0);
  }
  if (t < tiles && tid == 0) {          // gave up: the copies under way, of this tile and the next, land before the CTA leaves
    // (the tile's number from t: with n used here too the loop over 16-bit tiles came out a fifth slower)
    const int issued = static_cast<int>((t - blockIdx.x) / gridDim.x) + (t + static_cast<int64_t>(gridDim.x) < tiles ? 2 : 1);
    ring_drain(2, issued & 1, issued >> 1 & 1, [&](int s) { return smem_u32(&full_s[s]); });
  }
}

// Rows of any alignment: a CTA brings its tile into shared memory itself, and makes the codes along the rows from the
// registers on the way.
template <int DT>
__global__ void __launch_bounds__(kColThreads) mxfp4_cols_kernel(QuantParams p) {
  constexpr int EB = 4 / FloatTraits<DT>::kPerWord, kWords = 8 / FloatTraits<DT>::kPerWord;
  constexpr int kPasses = kTR * (kTC / 8) / kColThreads, kAhead = DT == BSIR_F32 ? 4 : kPasses;   // loads ahead of the first use
  constexpr int kStep = kColThreads / 8;                 // rows between a thread's vectors
  extern __shared__ __align__(16) uint8_t tile[];        // [kTR][kTC] elements, then [kTC][kCodeRow] codes
  uint8_t *codes_s = tile + kTR * kTC * EB;
  __shared__ uint8_t scale_s[kTC][kColPieces];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * kTR;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) * kTC;
  const int tid = threadIdx.x, r = tid >> 3, c = (tid & 7) * 8;
  const int rows = static_cast<int>(min(static_cast<int64_t>(kTR), p.rows - r0));       // of the tile
  const int nbytes = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(4), (p.cols - c0 - c + 1) / 2)));
  uint8_t *q = p.q + (r0 + r) * p.qs + (c0 + c) / 2, *s = p.s + (r0 + r) * p.ss + (c0 + c) / kBlock;
#pragma unroll
  for (int u0 = 0; u0 < kPasses; u0 += kAhead) {
    uint32_t w[kAhead][kWords];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int row = r + (u0 + u) * kStep;
      load8<DT, false>(p.x, (r0 + row) * p.xs, c0 + c, row < rows ? p.cols : 0, w[u]);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int row = r + (u0 + u) * kStep;
#pragma unroll
      for (int j = 0; j < kWords; j += 4)
        *reinterpret_cast<uint4 *>(tile + (row * kTC + c) * EB + 4 * j) = make_uint4(w[u][j], w[u][j + 1], w[u][j + 2], w[u][j + 3]);
      if (p.q) {
        uint32_t byte;
        const uint32_t codes = quant8<DT>(w[u], &byte);
        if (row < rows && nbytes > 0) {
          store_codes(q, codes, nbytes, p.q_words);
          if ((tid & 3) == 0) *s = static_cast<uint8_t>(byte);
        }
        q += kStep * p.qs;
        s += kStep * p.ss;
      }
    }
  }
  __syncthreads();
  quant_down<DT>(tile, codes_s, scale_s, tid >> 5);
  __syncthreads();
  store_down(p, codes_s, scale_s, r0, c0);
}

// codes and exponents -> values: a lane takes eight codes (4 bytes in, 16 or 32 bytes out)
struct DequantParams {
  int64_t cols;
  const uint8_t *q;
  int64_t qs;
  const uint8_t *s;
  int64_t ss;
  void *y;
  int64_t ys;
  FastDiv div;
  uint32_t nvec;
  int q_words;
};
// eight codes and their exponent byte -> eight elements as they lie in memory.  A code's magnitude bits, put at the
// bottom of bf16's exponent and top of its mantissa, are the value times 2^-126; two multiplications by powers of two
// (one would need 2^253) give the scaled value on pairs, exact down to bf16's subnormals.
template <int DT>
__device__ __forceinline__ void dequant8(uint32_t codes, uint32_t byte, uint32_t *w) {
  constexpr int kPer = FloatTraits<DT>::kPerWord;
  // 2^(byte - 127): byte 0 is 2^-127, under f32's normals (bits 0x00400000); 255 is NaN
  const uint32_t sc = byte == 255u ? 0x7fc00000u : byte == 0u ? 0x00400000u : byte << 23;
  if constexpr (DT == BSIR_BF16) {
    const uint32_t sc2 = sc | (sc >> 16);
    uint32_t t[4];                                  // elements i and i + 4
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t c = codes >> (4 * i);
      t[i] = mul_bf16x2(mul_bf16x2(((c << 6) & 0x01c001c0u) | ((c << 12) & 0x80008000u), 0x7e807e80u), sc2);
    }
    w[0] = __byte_perm(t[0], t[1], 0x5410);
    w[1] = __byte_perm(t[2], t[3], 0x5410);
    w[2] = __byte_perm(t[0], t[1], 0x7632);
    w[3] = __byte_perm(t[2], t[3], 0x7632);
  } else {
    float v[8];
    unpack_e2m1x8(codes, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], __uint_as_float(sc));
#pragma unroll
    for (int j = 0; j < 8 / kPer; ++j) w[j] = FloatTraits<DT>::pack(v + j * kPer);
  }
}
template <int DT, bool VEC, bool FLAT>
__global__ void __launch_bounds__(256) mxfp4_dequant_kernel(DequantParams p) {
  constexpr int kPer = FloatTraits<DT>::kPerWord, kWords = 8 / kPer;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t v0 = blockIdx.x * (256u * kRowVecs) + threadIdx.x;
  uint32_t codes[kRowVecs], byte[kRowVecs], row[kRowVecs], col[kRowVecs];
#pragma unroll
  for (int u = 0; u < kRowVecs; ++u) {
    const uint32_t i = v0 + u * 256u;
    codes[u] = byte[u] = row[u] = col[u] = 0;
    if constexpr (FLAT) {
      if (i < p.nvec) {
        codes[u] = reinterpret_cast<const uint32_t *>(p.q)[i];
        byte[u] = p.s[i >> 2];
      }
    } else {
      if (i >= p.nvec) continue;
      row[u] = fast_div(p.div, i);
      col[u] = (i - row[u] * p.div.d) * 8u;
      if (col[u] >= p.cols) continue;
      const uint8_t *src = p.q + static_cast<int64_t>(row[u]) * p.qs + col[u] / 2;
      const int nbytes = static_cast<int>(min(static_cast<int64_t>(4), (p.cols - col[u] + 1) / 2));
      if (p.q_words && nbytes == 4) {
        codes[u] = *reinterpret_cast<const uint32_t *>(src);
      } else {
        for (int j = 0; j < 4 && j < nbytes; ++j) codes[u] |= static_cast<uint32_t>(src[j]) << (8 * j);
      }
      byte[u] = p.s[static_cast<int64_t>(row[u]) * p.ss + col[u] / kBlock];
    }
  }
#pragma unroll
  for (int u = 0; u < kRowVecs; ++u) {
    const uint32_t i = v0 + u * 256u;
    const bool live = i < p.nvec && (FLAT || col[u] < p.cols);
    uint32_t w[kWords];
    dequant8<DT>(codes[u], byte[u], w);
    const int64_t at = FLAT ? static_cast<int64_t>(i) * 8 : static_cast<int64_t>(row[u]) * p.ys + col[u];
    if constexpr (VEC) {
      char *dst = static_cast<char *>(p.y) + at * (4 / kPer);
      if constexpr (FLAT && kWords == 8) {
        // 32 bytes a lane: neighbours swap halves, so that a store covers whole sectors (nvec is a multiple of 4: both
        // of a pair are here)
        const bool odd = threadIdx.x & 1;
        uint32_t a[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          a[j] = __shfl_xor_sync(0xffffffffu, odd ? w[j] : w[4 + j], 1);
        }
        const Vec16 mine{{odd ? w[4] : w[0], odd ? w[5] : w[1], odd ? w[6] : w[2], odd ? w[7] : w[3]}}, other{{a[0], a[1], a[2], a[3]}};
        if (live) {
          st_stream(odd ? dst - 16 : dst, odd ? other : mine);
          st_stream(odd ? dst + 16 : dst + 32, odd ? mine : other);
        }
      } else if (live) {
#pragma unroll
        for (int j = 0; j < kWords; j += 4) st_stream(dst + 4 * j, Vec16{{w[j], w[j + 1], w[j + 2], w[j + 3]}});
      }
    } else if (live) {
      for (int j = 0; j < 8 && col[u] + j < p.cols; ++j) {
        if constexpr (DT == BSIR_F32) static_cast<uint32_t *>(p.y)[at + j] = w[j];
        else static_cast<uint16_t *>(p.y)[at + j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
      }
    }
  }
}

template <int DT, bool VEC>
int32_t launch_quant(QuantParams p, cudaStream_t st) {
  if (p.qt) {
    constexpr int EB = DT == BSIR_F32 ? 4 : 2;
    const int64_t gx = ceil_div(p.cols, kTC), gy = ceil_div(p.rows, kTR);
    // the copy engine wants 16-byte aligned rows, byte coordinates and rows in 32 bits
    if (aligned_to(p.x, 16) && (p.xs * EB) % 16 == 0 && p.cols * EB <= 0x7fffffff && p.rows <= 0x7fffffff) {
      CUtensorMap map;
      int *err = device_error_word();
      if (!err) return fail(BSIR_ERR_WORKSPACE, "quant_mxfp4: no device error word");
      if (make_byte_tmap2(&map, p.x, p.cols * EB, p.rows, p.xs * EB, kTC * EB, kTR, p.q && DT != BSIR_F32)) {
        constexpr size_t smem = 2 * (kTR * kTC * EB + kTC * kCodeRow) + (EB == 2 ? 1024 : 128);
        const auto kernel = p.q ? mxfp4_cols_tma_kernel<DT, true> : mxfp4_cols_tma_kernel<DT, false>;
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        const int64_t sms = device_info().sm_count > 0 ? device_info().sm_count : 148, tiles = gx * gy;
        const int64_t ctas = sms * (DT == BSIR_F32 ? (p.q ? 3 : 2) : p.q ? 4 : 5);           // what shared memory holds
        launch_pdl(kernel, dim3(static_cast<unsigned>(tiles < ctas ? tiles : ctas)), dim3(p.q ? 2 * kColThreads : kColThreads), smem, st, map, p, tiles, gx, err);
        count_launch();
        return check_launch("quant_mxfp4");
      }
    }
    constexpr size_t smem = kTR * kTC * EB + kTC * kCodeRow;
    cudaFuncSetAttribute(mxfp4_cols_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    // The grid's y axis ends at 65535: longer matrices go in strips of rows (a strip starts at a whole block).
    for (int64_t y0 = 0; y0 < gy; y0 += 65535) {
      QuantParams s = p;
      const int64_t r0 = y0 * kTR, ny = gy - y0 < 65535 ? gy - y0 : 65535;
      s.x = static_cast<const char *>(p.x) + r0 * p.xs * EB;
      s.rows = p.rows - r0 < ny * kTR ? p.rows - r0 : ny * kTR;
      if (p.q) { s.q = p.q + r0 * p.qs; s.s = p.s + r0 * p.ss; }
      s.qt = p.qt + r0 / 2;
      s.st = p.st + r0 / kBlock;
      launch_pdl(mxfp4_cols_kernel<DT>, dim3(static_cast<unsigned>(gx), static_cast<unsigned>(ny)), dim3(kColThreads), smem, st, s);
      count_launch();
    }
    return check_launch("quant_mxfp4");
  }
  const int64_t vpr = ceil_div(p.cols, kBlock) * 4;
  const int64_t step = (int64_t{1} << 30) / vpr > 0 ? (int64_t{1} << 30) / vpr : 1;   // rows of one launch: 32-bit vector indices
  for (int64_t r = 0; r < p.rows; r += step) {
    QuantParams s = p;
    s.rows = p.rows - r < step ? p.rows - r : step;
    s.x = static_cast<const char *>(p.x) + r * p.xs * dtype_bytes(DT);
    s.q = p.q + r * p.qs;
    s.s = p.s + r * p.ss;
    s.div = make_fastdiv(static_cast<uint32_t>(vpr));
    s.nvec = static_cast<uint32_t>(s.rows * vpr);
    const dim3 grid(static_cast<unsigned>(ceil_div(s.nvec, 256 * kRowVecs)));
    if constexpr (VEC) {
      const bool flat = p.cols % kBlock == 0 && p.q_words && (p.rows == 1 || (p.xs == p.cols && p.qs == p.cols / 2 && p.ss == p.cols / kBlock));
      if (flat) launch_pdl(mxfp4_rows_kernel<DT, true, true>, grid, dim3(256), 0, st, s);
      else launch_pdl(mxfp4_rows_kernel<DT, true, false>, grid, dim3(256), 0, st, s);
    } else {
      launch_pdl(mxfp4_rows_kernel<DT, false, false>, grid, dim3(256), 0, st, s);
    }
    count_launch();
  }
  return check_launch("quant_mxfp4");
}
template <int DT, bool VEC>
int32_t launch_dequant(DequantParams p, int64_t rows, cudaStream_t st) {
  const int64_t vpr = ceil_div(p.cols, kBlock) * 4;
  const int64_t step = (int64_t{1} << 30) / vpr > 0 ? (int64_t{1} << 30) / vpr : 1;
  for (int64_t r = 0; r < rows; r += step) {
    DequantParams s = p;
    s.q = p.q + r * p.qs;
    s.s = p.s + r * p.ss;
    s.y = static_cast<char *>(p.y) + r * p.ys * dtype_bytes(DT);
    s.div = make_fastdiv(static_cast<uint32_t>(vpr));
    s.nvec = static_cast<uint32_t>((rows - r < step ? rows - r : step) * vpr);
    const dim3 grid(static_cast<unsigned>(ceil_div(s.nvec, 256 * kRowVecs)));
    if constexpr (VEC) {
      const bool flat = p.cols % kBlock == 0 && p.q_words && (rows == 1 || (p.ys == p.cols && p.qs == p.cols / 2 && p.ss == p.cols / kBlock));
      if (flat) launch_pdl(mxfp4_dequant_kernel<DT, true, true>, grid, dim3(256), 0, st, s);
      else launch_pdl(mxfp4_dequant_kernel<DT, true, false>, grid, dim3(256), 0, st, s);
    } else {
      launch_pdl(mxfp4_dequant_kernel<DT, false, false>, grid, dim3(256), 0, st, s);
    }
    count_launch();
  }
  return check_launch("dequant_mxfp4");
}

// [rows, cols] codes and exponents: strides and sizes (a 32-bit column index holds a row's vectors)
int32_t check_codes(const char *what, int64_t rows, int64_t cols, const void *q, int64_t qs, const void *s, int64_t ss) {
  if (!q || !s) return fail(BSIR_ERR_NULL, "%s: null pointer", what);
  if (rows > 1 && (qs < (cols + 1) / 2 || ss < ceil_div(cols, kBlock)))
    return fail(BSIR_ERR_STRIDE, "%s: row strides %lld / %lld bytes for %lld columns (codes take %lld, exponents %lld)", what, (long long)qs,
                (long long)ss, (long long)cols, (long long)((cols + 1) / 2), (long long)ceil_div(cols, kBlock));
  return BSIR_OK;
}
bool ranges_overlap(const void *a, int64_t na, const void *b, int64_t nb) {
  const char *a0 = static_cast<const char *>(a), *b0 = static_cast<const char *>(b);
  return a0 < b0 + nb && b0 < a0 + na;
}
// rows of bytes: `rows` stretches of `width`, `stride` apart
struct ByteRows {
  const uint8_t *p;
  int64_t rows, width, stride;
  int64_t span() const { return (rows - 1) * stride + width; }
};
// Whether two such sets share a byte.  Codes and exponents may lie side by side in rows of one buffer, so the stretches
// count, not the spans from the first to the last.
bool rows_overlap(ByteRows a, ByteRows b) {
  if (!ranges_overlap(a.p, a.span(), b.p, b.span())) return false;
  if (a.rows > b.rows) { const ByteRows t = a; a = b; b = t; }
  if (a.stride == b.stride) {                    // one place within a row's pitch for all rows
    const int64_t ahead = static_cast<int64_t>(reinterpret_cast<intptr_t>(b.p) - reinterpret_cast<intptr_t>(a.p));
    const int64_t d = ((ahead % a.stride) + a.stride) % a.stride;
    return d < a.width || d + b.width > a.stride;
  }
  for (int64_t i = 0; i < a.rows; ++i) {         // the first row of b that ends behind this one's start
    const int64_t at = static_cast<int64_t>(reinterpret_cast<intptr_t>(a.p) - reinterpret_cast<intptr_t>(b.p)) + i * a.stride;
    const int64_t j = at < b.width ? 0 : (at - b.width) / b.stride + 1;
    if (j < b.rows && j * b.stride < at + a.width) return true;
  }
  return false;
}

}  // namespace
}  // namespace bsir

using namespace bsir;

extern "C" int32_t bsir_quant_mxfp4(int32_t dtype, int64_t rows, int64_t cols, const void *x, int64_t x_row_stride, uint8_t *q,
                                    int64_t q_row_stride, uint8_t *scale, int64_t scale_row_stride, uint8_t *qt, int64_t qt_row_stride,
                                    uint8_t *scale_t, int64_t scale_t_row_stride, void *stream) {
  clear_error();
  if (!dtype_is_float(dtype)) return fail(BSIR_ERR_DTYPE, "quant_mxfp4: dtype %d (f32, f16, bf16)", dtype);
  if (rows < 0 || cols < 0 || rows > (int64_t{1} << 31) || cols > (int64_t{1} << 31))
    return fail(BSIR_ERR_SHAPE, "quant_mxfp4: [%lld, %lld] (at most 2^31 either way)", (long long)rows, (long long)cols);
  if ((q == nullptr) != (scale == nullptr) || (qt == nullptr) != (scale_t == nullptr))
    return fail(BSIR_ERR_NULL, "quant_mxfp4: codes and exponents of a direction come together");
  if (rows == 0 || cols == 0) return BSIR_OK;
  if (!x || (!q && !qt)) return fail(BSIR_ERR_NULL, "quant_mxfp4: null pointer");
  const int eb = dtype_bytes(dtype);
  if (rows > 1 && x_row_stride < cols) return fail(BSIR_ERR_STRIDE, "quant_mxfp4: row stride %lld of %lld columns", (long long)x_row_stride, (long long)cols);
  if (!aligned_to(x, eb)) return fail(BSIR_ERR_ALIGN, "quant_mxfp4: misaligned");
  if (rows == 1) { x_row_stride = cols; q_row_stride = (cols + 1) / 2; scale_row_stride = ceil_div(cols, kBlock); }
  if (cols == 1) { qt_row_stride = (rows + 1) / 2; scale_t_row_stride = ceil_div(rows, kBlock); }
  const int64_t x_bytes = ((rows - 1) * x_row_stride + cols) * eb;
  for (int d = 0; d < 2; ++d) {
    const void *cq = d ? qt : q, *cs = d ? scale_t : scale;
    if (!cq) continue;
    const int64_t r = d ? cols : rows, c = d ? rows : cols, qs = d ? qt_row_stride : q_row_stride, ss = d ? scale_t_row_stride : scale_row_stride;
    if (int32_t rc = check_codes("quant_mxfp4", r, c, cq, qs, cs, ss)) return rc;
    if (ranges_overlap(x, x_bytes, cq, (r - 1) * qs + (c + 1) / 2) || ranges_overlap(x, x_bytes, cs, (r - 1) * ss + ceil_div(c, kBlock)))
      return fail(BSIR_ERR_UNSUPPORTED, "quant_mxfp4: a result may not overlap the source");
  }
  const ByteRows results[4] = {{q, rows, (cols + 1) / 2, q_row_stride}, {scale, rows, ceil_div(cols, kBlock), scale_row_stride},
                               {qt, cols, (rows + 1) / 2, qt_row_stride}, {scale_t, cols, ceil_div(rows, kBlock), scale_t_row_stride}};
  for (int i = 0; i < 4; ++i)
    for (int j = i + 1; j < 4; ++j)
      if (results[i].p && results[j].p && rows_overlap(results[i], results[j]))
        return fail(BSIR_ERR_UNSUPPORTED, "quant_mxfp4: the results may not overlap each other");
  QuantParams p{};
  p.rows = rows; p.cols = cols; p.x = x; p.xs = x_row_stride;
  p.q = q; p.qs = q_row_stride; p.s = scale; p.ss = scale_row_stride;
  p.qt = qt; p.qts = qt_row_stride; p.st = scale_t; p.sts = scale_t_row_stride;
  p.q_words = q && aligned_to(q, 4) && q_row_stride % 4 == 0;
  p.qt_words = qt && aligned_to(qt, 16) && qt_row_stride % 16 == 0;
  const bool vec = cols % 8 == 0 && aligned_to(x, 16) && (x_row_stride * eb) % 16 == 0;
  cudaStream_t st = resolve_stream(stream);
  switch (dtype) {
    case BSIR_F32: return vec ? launch_quant<BSIR_F32, true>(p, st) : launch_quant<BSIR_F32, false>(p, st);
    case BSIR_F16: return vec ? launch_quant<BSIR_F16, true>(p, st) : launch_quant<BSIR_F16, false>(p, st);
    default: return vec ? launch_quant<BSIR_BF16, true>(p, st) : launch_quant<BSIR_BF16, false>(p, st);
  }
}

extern "C" int32_t bsir_dequant_mxfp4(int32_t dtype, int64_t rows, int64_t cols, const uint8_t *q, int64_t q_row_stride, const uint8_t *scale,
                                      int64_t scale_row_stride, void *y, int64_t y_row_stride, void *stream) {
  clear_error();
  if (!dtype_is_float(dtype)) return fail(BSIR_ERR_DTYPE, "dequant_mxfp4: dtype %d (f32, f16, bf16)", dtype);
  if (rows < 0 || cols < 0 || rows > (int64_t{1} << 31) || cols > (int64_t{1} << 31))
    return fail(BSIR_ERR_SHAPE, "dequant_mxfp4: [%lld, %lld] (at most 2^31 either way)", (long long)rows, (long long)cols);
  if (rows == 0 || cols == 0) return BSIR_OK;
  if (!y) return fail(BSIR_ERR_NULL, "dequant_mxfp4: null pointer");
  if (int32_t rc = check_codes("dequant_mxfp4", rows, cols, q, q_row_stride, scale, scale_row_stride)) return rc;
  if (rows > 1 && y_row_stride < cols) return fail(BSIR_ERR_STRIDE, "dequant_mxfp4: row stride %lld of %lld columns", (long long)y_row_stride, (long long)cols);
  const int eb = dtype_bytes(dtype);
  if (!aligned_to(y, eb)) return fail(BSIR_ERR_ALIGN, "dequant_mxfp4: misaligned");
  if (rows == 1) { q_row_stride = (cols + 1) / 2; scale_row_stride = ceil_div(cols, kBlock); y_row_stride = cols; }
  const int64_t y_bytes = ((rows - 1) * y_row_stride + cols) * eb;
  if (ranges_overlap(y, y_bytes, q, (rows - 1) * q_row_stride + (cols + 1) / 2) ||
      ranges_overlap(y, y_bytes, scale, (rows - 1) * scale_row_stride + ceil_div(cols, kBlock)))
    return fail(BSIR_ERR_UNSUPPORTED, "dequant_mxfp4: the result may not overlap the source");
  DequantParams p{};
  p.cols = cols; p.q = q; p.qs = q_row_stride; p.s = scale; p.ss = scale_row_stride; p.y = y; p.ys = y_row_stride;
  p.q_words = aligned_to(q, 4) && q_row_stride % 4 == 0;
  const bool vec = cols % 8 == 0 && aligned_to(y, 16) && (y_row_stride * eb) % 16 == 0;
  cudaStream_t st = resolve_stream(stream);
  switch (dtype) {
    case BSIR_F32: return vec ? launch_dequant<BSIR_F32, true>(p, rows, st) : launch_dequant<BSIR_F32, false>(p, rows, st);
    case BSIR_F16: return vec ? launch_dequant<BSIR_F16, true>(p, rows, st) : launch_dequant<BSIR_F16, false>(p, rows, st);
    default: return vec ? launch_dequant<BSIR_BF16, true>(p, rows, st) : launch_dequant<BSIR_BF16, false>(p, rows, st);
  }
}
