// mxfp4_gemm.cu -- products of microscaled 4-bit matrices (MXFP4, see mxfp4_quant.cu) on the tensor core:
//   C[i, j] = cast_rint( sum_k A[i, k] * B[j, k] + bias[j] ),   A[i, k] = code * 2^(exponent byte of (i, k / 32) - 127)
// for one B, or row groups of A against a B of their own (the experts' products of a mixture-of-experts layer: rows
// offsets[e] .. offsets[e + 1] of A meet B[e]; other rows of C are left as they were).
//
// tcgen05.mma kind::mxf4.block_scale multiplies 64 elements of K an instruction and applies both exponents on the way
// into the f32 accumulator, four times the rate of a 16-bit product.  Codes come by TMA into 128-byte-swizzled tiles
// (a 128-byte row is 256 elements of K); the exponents have to lie in tensor memory: row r of an operand tile at lane
// r % 32, column r / 32, four bytes (128 elements of K) a cell, the same in all four lane quadrants.  The exponent
// matrices keep the plain [rows, K / 32] layout, so groups may start at any row: TMA brings [rows x 32 bytes] (1024
// elements of K; 16 bytes a row moved half-empty sectors and cost 4 to 9 %), warps turn them in shared memory from a row's
// eight words into a lane's four rows, and the MMA issuer copies them to tensor memory with tcgen05.cp ahead of the
// instructions that use them, in order and without a barrier between.
//
// What bounds it (B200, 4096 x 14336 x 4096): one more tile a pair takes 6.6 us, of which 16 stages at 0.36 us (512 cycles
// of multiplication each, 0.27) and 0.8 for the accumulator's way out; the tensor pipe is active 68 % of the launch, and 46
// of the 64 bytes a cycle that reach an SM come from L2.  Sustained, the board's power limit lowers the clock to 1.5 GHz: 92 us
// when cool, 113 sustained (4.3 PFLOP/s).  Up to 32 rows the weights' way from HBM bounds it.
//
// A persistent kernel, one CTA per SM, 256 threads (384 with one accumulator):
//   warp 0            TMA producer of codes (a ring of stages of 256 elements of K) and exponents (a ring of 1024)
//   warp 1            issuer of tcgen05.cp and tcgen05.mma
//   warps 2-5 (2-9)   epilogue: accumulator -> bias -> rounding -> C
//   the last two      exponents: rows of eight words -> lanes of four rows, 128 rows at a time
// in three forms:
//   kPair    256 rows of A x BN columns of C on two CTAs (cta_group::2): each holds its 128 rows of A and half of the
//            tile's rows of B, so that an SM's shared memory is read and filled for B half as often;
//   kSingle  128 rows x BN columns on one CTA, for groups that would leave much of a 256-row tile empty;
//   kFew     operands swapped: 128 rows of B are the instruction's M side and BN rows of A its N side, so that weights
//            are streamed for as few as 16 rows of A.
// With few tiles a cluster of up to eight CTAs shares the K of a tile of kSingle or kFew, and has that tile only: each CTA
// leaves its part in shared memory and adds its share of the rows from all of them, in their order (the same bits on every
// run of a device; how many share it goes by how many clusters the device runs at once).  64 x 4096 x 14336: 11.3 us, 18.8
// whole; 1 x 2048 x 8192: 6.4, 11 whole.  (Parts handed over by asynchronous
// stores straight from tensor memory cost 0.6 to 2 us more: eight bytes each, and more instructions to fetch.)
#include "tc_ptx.cuh"

#include <atomic>

namespace bsir {
namespace {

constexpr int kTileM = 128;
constexpr int kStageK = 256;       // elements of K a stage: one 128-byte swizzle row of codes
constexpr int kChunk = 4;           // stages that a piece of exponents lasts: 32 bytes (a sector) of each row
constexpr int kMaxGroups = 1024;
enum MxMode { kSingle, kPair, kFew };

struct MxParams {
  int64_t m, n;
  int k_blocks;                    // stages of a tile
  const int32_t *offsets;          // [groups + 1] or null: one group of all rows
  int groups;
  const void *bias;
  int64_t bias_stride;             // elements between the groups' biases
  int32_t bias_dtype, out_dtype;
  void *out;
  int64_t ldo;
  int *err;
  int tma_out;                     // 1: C's rows start 16-byte aligned (TMA stores, 16-byte pieces)
  int split;                       // CTAs that work on a tile: those that share its K (kFew, kSingle), two of kPair
};

template <int BN, int MODE>
struct MxCfg {
  static constexpr int kNRows = MODE == kPair ? BN / 2 : BN;         // rows of the N side's codes in this CTA
  static constexpr int kStage = (kTileM + kNRows) * 128;
  static constexpr int kSfBlocks = 1 + (BN + 127) / 128;             // blocks of 128 rows of exponents: M side, N side
  static constexpr int kSfStage = kSfBlocks * 4096;
  static constexpr int kSfStages = 2;
  static constexpr int kAccs = BN > 192 ? 1 : 2;
  // columns of tensor memory: accumulators, then each stage's exponents: two words (128 elements of K each) of four
  // columns a block, the N side's first
  static constexpr int kSfN = (kSfBlocks - 1) * 4;
  static constexpr int kSfCols = 2 * (kSfN + 4);
  static constexpr int kSfBase = kAccs * BN;
  static constexpr int kSfBufs = (512 - kSfBase) / kSfCols;
  // staging: one or two buffers of 32 rows x 128 bytes of C a warp, or a tile
  static constexpr int kEpiWarps = kAccs == 1 ? 8 : 4;               // two a lane quadrant share the columns of a lone accumulator
  static constexpr int kEpiBufs = kAccs == 1 ? 1 : 2;
  static constexpr int kThreads = 128 + 32 * kEpiWarps;
  static constexpr int kEpi = MODE == kFew ? BN * kTileM * 4 : kEpiWarps * kEpiBufs * 4096;
  static constexpr int kTable = 2 * (kMaxGroups + 1) * 4;
  static constexpr int kFixed = kSfStages * kSfStage + kEpi + 512 /*barriers*/ + kTable + 1024 /*alignment*/;
  static constexpr int kFit = (227 * 1024 - kFixed) / kStage;
  static constexpr int kMost = kSfBufs < 9 ? kSfBufs : 9;
  static constexpr int kStages = kFit > kMost ? kMost : kFit;
  static constexpr int kCols = kSfBase + kStages * kSfCols;
  static constexpr int kTmemCols = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static constexpr int kSfOff = kStages * kStage;
  static constexpr int kEpiOff = kSfOff + kSfStages * kSfStage;    // 128-byte swizzle
  static constexpr int kBarOff = kEpiOff + kEpi;
  static constexpr int kTableOff = kBarOff + 512;                    // tiles before a group, first row of a group
  static constexpr int kSmem = kTableOff + kTable + 1024;
  static_assert(kCols <= 512, "tensor memory");
  static_assert(kStages >= 4 && kSmem <= 227 * 1024, "shared memory");
  static_assert(kStages * kStage >= (MODE == kFew ? BN : kTileM) * 128 * 4, "the ring holds a partial tile");
};

// The issuing warp's instructions.  All 32 lanes execute them and the predicate of one elected lane lets them through:
// without a branch around them their operands are warp-uniform values, and one issues every 68 to 73 cycles, under the
// 96 to 128 that the tensor core takes for N = 192 to 256; behind a branch (one lane of the warp, elected or lane 0)
// it was 97 to 167.  Shared-memory descriptors come as their low words (address / 16); the high word is the same for
// every K-major tile with the 128-byte swizzle (8-row groups 1024 bytes apart, version 1).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr) { return (saddr >> 4) | (1u << 16); }
template <int MODE>
__device__ __forceinline__ void mma_mxf4(uint32_t elected, uint32_t tmem_d, uint32_t adesc, uint32_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
  if constexpr (MODE == kPair) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 e, %8, 0;\n\t"
        "mov.b64 a, {%1, %7};\n\tmov.b64 b, {%2, %7};\n\t"
        "@e tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d),
        "r"(adesc), "r"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "n"(kDescHi), "r"(elected)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 e, %8, 0;\n\t"
        "mov.b64 a, {%1, %7};\n\tmov.b64 b, {%2, %7};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d),
        "r"(adesc), "r"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "n"(kDescHi), "r"(elected)
        : "memory");
  }
}
// 32 lanes x 16 bytes of shared memory (no swizzle, 8 rows of 16 bytes 128 bytes apart) -> four columns of tensor
// memory, repeated in the four lane quadrants; cta_group::2: in both CTAs, each from its own shared memory
constexpr uint32_t kCopyDescHi = (128u >> 4) | (1u << 14);
template <int MODE>
__device__ __forceinline__ void tmem_copy(uint32_t elected, uint32_t taddr, uint32_t saddr) {
  if constexpr (MODE == kPair)
    asm volatile(
        "{\n\t.reg .pred e;\n\t.reg .b64 a;\n\tsetp.ne.b32 e, %2, 0;\n\tmov.b64 a, {%1, %3};\n\t"
        "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], a;\n\t}" ::"r"(taddr),
        "r"(saddr >> 4), "r"(elected), "n"(kCopyDescHi)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred e;\n\t.reg .b64 a;\n\tsetp.ne.b32 e, %2, 0;\n\tmov.b64 a, {%1, %3};\n\t"
        "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], a;\n\t}" ::"r"(taddr),
        "r"(saddr >> 4), "r"(elected), "n"(kCopyDescHi)
        : "memory");
}
template <int MODE>
__device__ __forceinline__ void commit_to(uint32_t elected, uint32_t bar) {   // kPair: the barrier of both CTAs
  if constexpr (MODE == kPair)
    asm volatile(
        "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}" ::"r"(bar),
        "r"(elected), "h"(static_cast<uint16_t>(3))
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(elected)
        : "memory");
}
template <bool CLUSTER>
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {      // without waiting
  uint32_t done;
  if constexpr (CLUSTER)
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
// e2m1 x e2m1, exponents E8M0, both K-major; `sf_id` (0 or 2): which two of a cell's four bytes belong to these 64
// elements of K
__device__ __forceinline__ uint32_t mx_idesc(int n, int m, uint32_t sf_id) {
  return (sf_id << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(m >> 7) << 27) | (sf_id << 29);
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(leader_bar)
      : "memory");
}
// Arrival on a barrier of the pair's leader by a thread that hands over its own CTA's shared memory (made visible to the
// tensor core by fence.proxy.async) or tensor memory (ordered by tcgen05.fence).  The release at cluster scope is restricted
// to shared memory: the arrival's own, of everything, took about 1400 cycles next to running copies.
__device__ __forceinline__ void mbar_arrive_leader(uint32_t cluster_addr) {
  asm volatile("fence.release.sync_restrict::shared::cta.cluster;" ::: "memory");
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {       // 1 in one lane of the (whole) warp
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one;
}

__device__ __forceinline__ float load_float(const void *p, int32_t dtype, int64_t i) {
  if (dtype == BSIR_F32) return static_cast<const float *>(p)[i];
  const unsigned short h = static_cast<const unsigned short *>(p)[i];
  return dtype == BSIR_F16 ? __half2float(__ushort_as_half(h)) : __uint_as_float(static_cast<uint32_t>(h) << 16);
}
__device__ __forceinline__ void store_out(const MxParams &p, int64_t at, float f) {
  if (p.out_dtype == BSIR_F32) static_cast<float *>(p.out)[at] = f;
  else if (p.out_dtype == BSIR_F16) static_cast<__half *>(p.out)[at] = __float2half_rn(f);
  else static_cast<__nv_bfloat16 *>(p.out)[at] = __float2bfloat16_rn(f);
}

// Where a tile lies: `tile_start[g]` tiles come before group g, whose rows begin at row_start[g]; within a group the
// row tiles run fastest, so that CTAs working at the same time share rows of B.
struct MxTile {
  int group, row0, row_end, n0;
};
template <int ROWS, int COLS>
__device__ __forceinline__ void find_tile(int tile, const int *tile_start, const int *row_start, int &group, MxTile &t) {
  while (tile >= tile_start[group + 1]) ++group;            // a role's tiles only go up
  const int first = row_start[group], end = row_start[group + 1];
  const int row_tiles = (end - first + ROWS - 1) / ROWS;
  const int local = tile - tile_start[group];
  t.group = group;
  t.row0 = first + (local % row_tiles) * ROWS;
  t.row_end = end;
  t.n0 = (local / row_tiles) * COLS;
}

// 32 columns of an epilogue warp's 32 rows from tensor memory, bias added
__device__ __forceinline__ void load_columns(const MxParams &p, uint32_t acc, int group, int64_t col0, int lane, uint32_t *r) {
  tmem_ld32(acc, r);
  tmem_ld_wait();
  if (p.bias) {
    const int64_t col = col0 + lane;
    const float mine = col < p.n ? load_float(p.bias, p.bias_dtype, group * p.bias_stride + col) : 0.0f;
#pragma unroll
    for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__fadd_rn(__uint_as_float(r[j]), __shfl_sync(0xffffffffu, mine, j)));
  }
}
__device__ __forceinline__ void round_columns(const MxParams &p, const uint32_t *r, uint32_t *w) {
  if (p.out_dtype == BSIR_F16) {
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j] = pack_f16x2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j] = pack_bf16x2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
  }
}
// 64 bytes (half of a 128-byte piece) of this lane's row into the staging buffer, 128-byte swizzle
__device__ __forceinline__ void stage_half(uint8_t *row, int lane, int half, const uint32_t *w) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *reinterpret_cast<uint4 *>(row + (((4 * half + c) ^ (lane & 7)) * 16)) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
}

// An epilogue warp's 32 rows of C, 128 bytes a row at a time: staged in shared memory and sent by a TMA store; where
// that cannot be (rows behind the group's end in the box, C's rows not 16-byte aligned, a last piece of other than whole 16
// bytes) the warp stores them itself, row by row.
template <int BUFS> struct RowWriter {
  const MxParams &p;
  const CUtensorMap *tmap_out;
  const MxTile &t;
  int row0, lane, eb, rows;
  bool by_tma;
  uint8_t *stage;
  uint32_t stage_addr;
  uint32_t &nstores;
  __device__ __forceinline__ RowWriter(const MxParams &p_, const CUtensorMap *m, const MxTile &t_, int row0_, int lane_, uint8_t *stage_, uint32_t addr, uint32_t &n)
      : p(p_), tmap_out(m), t(t_), row0(row0_), lane(lane_), stage(stage_), stage_addr(addr), nstores(n) {
    eb = p.out_dtype == BSIR_F32 ? 4 : 2;
    rows = t.row_end - row0 < 32 ? t.row_end - row0 : 32;
    by_tma = p.tma_out && (rows == 32 || t.row_end == p.m);     // behind the last row of C nothing is written
  }
  // the buffer for the next piece: this lane's row of it
  __device__ __forceinline__ uint8_t *begin() {
    // the store that last used it has read it (it may have been an earlier tile's)
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(BUFS - 1) : "memory");
    __syncwarp();
    return stage + nstores % BUFS * 4096 + lane * 128;
  }
  __device__ __forceinline__ void send(int64_t col0, int cols) {     // `cols` of C from col0 on, at most 128 bytes
    uint8_t *buf = stage + nstores % BUFS * 4096;
    const int have = static_cast<int>(p.n - col0 < cols ? p.n - col0 : cols) * eb;    // bytes of a row
    // (a TMA store writes whole 16-byte pieces, whatever the map's extent and type: up to 15 bytes behind C's last column)
    if (by_tma && have % 16 == 0) {
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) tma_store_2d(tmap_out, static_cast<int>(col0) * eb, row0, stage_addr + nstores % BUFS * 4096);
      ++nstores;
      return;
    }
    __syncwarp();
    if (p.tma_out) {                                       // eight lanes a row, four rows at a time, sixteen in flight
      const int piece = lane & 7;
      if (have == 128) {
        char *dst = static_cast<char *>(p.out) + ((row0 + (lane >> 3)) * p.ldo + col0) * eb + piece * 16;
        const int64_t pitch = 4 * p.ldo * eb;
        for (int r0 = lane >> 3; r0 < rows; r0 += 16) {
          uint4 v[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const uint4 *>(buf + (r0 + 4 * u) * 128 + ((piece ^ ((r0 + 4 * u) & 7)) * 16));
#pragma unroll
          for (int u = 0; u < 4; ++u, dst += pitch)
            if (r0 + 4 * u < rows) *reinterpret_cast<uint4 *>(dst) = v[u];
        }
        __syncwarp();
        return;
      }
      for (int r = lane >> 3; r < rows; r += 4) {
        const uint4 v = *reinterpret_cast<const uint4 *>(buf + r * 128 + ((piece ^ (r & 7)) * 16));
        char *dst = static_cast<char *>(p.out) + ((row0 + r) * p.ldo + col0) * eb + piece * 16;
        if (piece * 16 + 16 <= have) {
          *reinterpret_cast<uint4 *>(dst) = v;
        } else {
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (piece * 16 + 2 * i < have) reinterpret_cast<uint16_t *>(dst)[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
        }
      }
    } else {
      // four bytes a lane, eight rows in flight (16-bit rows that are here whole ask nothing on the way: 333 x 5001 x 2900
      // 11.6 -> 10.6 us; words of two lanes' halves, stored whole, 14.7)
      const int at = lane * 4;
      const bool low = at < have, high = at + 2 < have;
      char *dst = static_cast<char *>(p.out) + (static_cast<int64_t>(row0) * p.ldo + col0) * eb + at;
      const int64_t pitch = p.ldo * eb;
      for (int r0 = 0; r0 < rows; r0 += 8) {
        uint32_t v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = *reinterpret_cast<const uint32_t *>(buf + (r0 + r) * 128 + (((at >> 4) ^ r) * 16) + (at & 15));
        if (have == 128 && r0 + 8 <= rows && eb == 2) {              // all of it: nothing to ask a row
          char *d = dst + r0 * pitch;
#pragma unroll
          for (int r = 0; r < 8; ++r, d += pitch) {
            reinterpret_cast<uint16_t *>(d)[0] = static_cast<uint16_t>(v[r]);
            reinterpret_cast<uint16_t *>(d)[1] = static_cast<uint16_t>(v[r] >> 16);
          }
          continue;
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          if (r0 + r >= rows || !low) continue;
          char *d = dst + (r0 + r) * pitch;
          if (eb == 4) {
            *reinterpret_cast<uint32_t *>(d) = v[r];
          } else {
            *reinterpret_cast<uint16_t *>(d) = static_cast<uint16_t>(v[r]);
            if (high) *reinterpret_cast<uint16_t *>(d + 2) = static_cast<uint16_t>(v[r] >> 16);
          }
        }
      }
    }
    __syncwarp();
  }
};

// One accumulator -> C.  `release()` hands the accumulator back to the issuer.  With a second accumulator the issuer is
// busy meanwhile and the columns go out as they come; with one (BN = 256) it is waiting: the warp's columns are first
// taken into registers whole.
// (BN columns from n0 on are this warp's; acc is their first.)
template <int BN, bool kDrain, class Writer, class Release>
__device__ __forceinline__ void store_rows(const MxParams &p, Writer &out, uint32_t acc, int group, int n0, int lane, Release release) {
  if (p.out_dtype == BSIR_F32) {
    if constexpr (kDrain) {
      uint32_t r[BN];
#pragma unroll
      for (int c = 0; c < BN; c += 32) tmem_ld32(acc + static_cast<uint32_t>(c), r + c);
      tmem_ld_wait();
      release();
      if (p.bias) {
        const float4 *bias = reinterpret_cast<const float4 *>(out.stage);
#pragma unroll
        for (int j = 0; j < BN / 4; ++j) {
          const float4 b = bias[j];
          r[4 * j] = __float_as_uint(__fadd_rn(__uint_as_float(r[4 * j]), b.x));
          r[4 * j + 1] = __float_as_uint(__fadd_rn(__uint_as_float(r[4 * j + 1]), b.y));
          r[4 * j + 2] = __float_as_uint(__fadd_rn(__uint_as_float(r[4 * j + 2]), b.z));
          r[4 * j + 3] = __float_as_uint(__fadd_rn(__uint_as_float(r[4 * j + 3]), b.w));
        }
      }
#pragma unroll
      for (int c = 0; c < BN; c += 32) {
        if (n0 + c >= p.n) break;
        uint8_t *row = out.begin();
        stage_half(row, lane, 0, r + c);
        stage_half(row, lane, 1, r + c + 16);
        out.send(n0 + c, 32);
      }
    } else {
      for (int c0 = 0; c0 < BN && n0 + c0 < p.n; c0 += 32) {
        uint32_t r[32];
        load_columns(p, acc + static_cast<uint32_t>(c0), group, n0 + c0, lane, r);
        uint8_t *row = out.begin();
        stage_half(row, lane, 0, r);
        stage_half(row, lane, 1, r + 16);
        out.send(n0 + c0, 32);
      }
      release();
    }
  } else if constexpr (kDrain) {
    uint32_t w[BN / 2];
    const float4 *bias = reinterpret_cast<const float4 *>(out.stage);     // put there before the accumulator was waited for
#pragma unroll
    for (int c = 0; c < BN / 64; ++c) {
      uint32_t r[64];
      tmem_ld32(acc + static_cast<uint32_t>(64 * c), r);
      tmem_ld32(acc + static_cast<uint32_t>(64 * c + 32), r + 32);
      tmem_ld_wait();
      if (p.bias) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float4 b = bias[16 * c + j];
          r[4 * j] = __float_as_uint(__fadd_rn(__uint_as_float(r[4 * j]), b.x));
          r[4 * j + 1] = __float_as_uint(__fadd_rn(__uint_as_float(r[4 * j + 1]), b.y));
          r[4 * j + 2] = __float_as_uint(__fadd_rn(__uint_as_float(r[4 * j + 2]), b.z));
          r[4 * j + 3] = __float_as_uint(__fadd_rn(__uint_as_float(r[4 * j + 3]), b.w));
        }
      }
      round_columns(p, r, w + 32 * c);
      round_columns(p, r + 32, w + 32 * c + 16);
    }
    release();
#pragma unroll
    for (int c = 0; c < BN / 64; ++c) {
      if (n0 + 64 * c >= p.n) break;
      uint8_t *row = out.begin();
      stage_half(row, lane, 0, w + 32 * c);
      stage_half(row, lane, 1, w + 32 * c + 16);
      out.send(n0 + 64 * c, 64);
    }
  } else {
    for (int c0 = 0; c0 < BN && n0 + c0 < p.n; c0 += 64) {
      uint32_t r[32], w[16];
      load_columns(p, acc + static_cast<uint32_t>(c0), group, n0 + c0, lane, r);
      round_columns(p, r, w);
      uint8_t *row = out.begin();
      stage_half(row, lane, 0, w);
      load_columns(p, acc + static_cast<uint32_t>(c0 + 32), group, n0 + c0 + 32, lane, r);
      round_columns(p, r, w);
      stage_half(row, lane, 1, w);
      out.send(n0 + c0, 64);
    }
    release();
  }
}

// A tile whose K is shared by a cluster: each CTA leaves its part [rows][128] of f32 in its ring of stages (16-byte
// pieces permuted within a row, so that neither a column of pieces nor a row meets in one bank), and after a cluster
// barrier each reads its share of the rows that C has from all of them and adds in the order of the CTAs.
template <int BN> __device__ __forceinline__ void store_partial(uint8_t *ring, uint32_t acc, int row) {
#pragma unroll
  for (int c0 = 0; c0 < BN; c0 += 32) {
    uint32_t r[32];
    tmem_ld32(acc + static_cast<uint32_t>(c0), r);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<uint4 *>(ring + row * (BN * 4) + (((c0 / 4 + j) ^ (row & 7)) * 16)) = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
  }
}
// the same of a tile whose operands were swapped: lane = column of C
template <int BN> __device__ __forceinline__ void store_partial_swapped(uint8_t *ring, uint32_t acc, int col) {
#pragma unroll
  for (int c0 = 0; c0 < BN; c0 += 16) {
    uint32_t r[16];
    tmem_ld16(acc + static_cast<uint32_t>(c0), r);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int row = c0 + j;
      *reinterpret_cast<uint32_t *>(ring + row * (kTileM * 4) + (((col >> 2) ^ (row & 7)) * 16) + (col & 3) * 4) = r[j];
    }
  }
}
__device__ __forceinline__ float4 load_peer4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
  return v;
}
// four neighbouring columns of C
__device__ __forceinline__ void load_bias4(const MxParams &p, int group, int64_t col, float *bias) {
#pragma unroll
  for (int i = 0; i < 4; ++i) bias[i] = p.bias && col + i < p.n ? load_float(p.bias, p.bias_dtype, group * p.bias_stride + col + i) : 0.0f;
}
__device__ __forceinline__ void store_piece(const MxParams &p, int64_t row, int64_t col, float4 sum, const float *bias) {
  const int64_t at = row * p.ldo + col;
  const float f[4] = {__fadd_rn(sum.x, bias[0]), __fadd_rn(sum.y, bias[1]), __fadd_rn(sum.z, bias[2]), __fadd_rn(sum.w, bias[3])};
  if (p.tma_out && col + 4 <= p.n) {
    if (p.out_dtype == BSIR_F32) {
      *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
      const uint2 w = p.out_dtype == BSIR_F16 ? make_uint2(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]))
                                              : make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
      *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + at) = w;
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < 4 && col + i < p.n; ++i) store_out(p, at + i, f[i]);
  }
}
template <int ROWS, int THREADS, int TEAM>
__device__ __forceinline__ void join_partials(const MxParams &p, const MxTile &t, uint32_t ring, int rank) {
  constexpr int kPieces = 32, kShare = ROWS / TEAM, kStep = THREADS / kPieces, kRows = (kShare + kStep - 1) / kStep;   // a thread's rows
  const int piece = threadIdx.x % kPieces, first = rank + threadIdx.x / kPieces * TEAM;      // every TEAM-th row is this CTA's
  if (first >= ROWS) return;
  float4 v[TEAM][kRows];
#pragma unroll
  for (int c = 0; c < TEAM; ++c) {                      // all of a thread's parts are on their way before the first is added
    const uint32_t peer = map_to_cta(ring, c);
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int row = first + u * (kStep * TEAM);
      if (t.row0 + row < t.row_end) v[c][u] = load_peer4(peer + static_cast<uint32_t>(row * (kTileM * 4) + ((piece ^ (row & 7)) * 16)));
    }
  }
  const int64_t col = t.n0 + 4 * piece;
  float bias[4];
  load_bias4(p, t.group, col, bias);
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int row = first + u * (kStep * TEAM);
    float4 sum = v[0][u];
#pragma unroll
    for (int c = 1; c < TEAM; ++c) {
      sum.x += v[c][u].x;
      sum.y += v[c][u].y;
      sum.z += v[c][u].z;
      sum.w += v[c][u].w;
    }
    if (t.row0 + row >= t.row_end) break;               // rows go up
    store_piece(p, t.row0 + row, col, sum, bias);
  }
}

template <int BN, int MODE>
__global__ void __launch_bounds__(MxCfg<BN, MODE>::kThreads, 1)
    mxfp4_gemm_kernel(const __grid_constant__ CUtensorMap tmap_m, const __grid_constant__ CUtensorMap tmap_n,
                      const __grid_constant__ CUtensorMap tmap_sm, const __grid_constant__ CUtensorMap tmap_sn,
                      const __grid_constant__ CUtensorMap tmap_out, MxParams p) {
  using Cfg = MxCfg<BN, MODE>;
  constexpr bool SWAP = MODE == kFew, PAIR = MODE == kPair;
  constexpr int kRows = SWAP ? BN : PAIR ? 2 * kTileM : kTileM;       // rows of A and columns of C (rows of B) a tile
  constexpr int kColsC = SWAP ? kTileM : BN;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t *gen = smem_raw + (base - raw);
  const uint32_t bars = base + Cfg::kBarOff;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (Cfg::kStages + s); };
  auto sf_full_bar = [&](int s) { return bars + 8u * (2 * Cfg::kStages + s); };
  auto sf_empty_bar = [&](int s) { return bars + 8u * (2 * Cfg::kStages + Cfg::kSfStages + s); };
  constexpr int kB2 = 2 * Cfg::kStages + 2 * Cfg::kSfStages;
  auto sf_ready_bar = [&](int s) { return bars + 8u * (kB2 + s); };                       // exponents turned
  constexpr int kB3 = kB2 + Cfg::kSfStages;
  auto acc_full_bar = [&](int b) { return bars + 8u * (kB3 + b); };
  auto acc_empty_bar = [&](int b) { return bars + 8u * (kB3 + 2 + b); };
  static_assert(8 * (kB3 + 4) + 16 <= 512, "barriers");
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(gen + Cfg::kBarOff + 8 * (kB3 + 4));
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);    // in a pair two counts of loads follow
  int *tile_start = reinterpret_cast<int *>(gen + Cfg::kTableOff);         // [groups + 1]
  int *row_start = tile_start + kMaxGroups + 1;                            // [groups + 1]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // CTAs that work on one tile: a pair (rows cut in two), or those that share its K (a cluster with one tile, or one CTA)
  const int team = PAIR ? 2 : p.split;
  const int rank = team > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int first_tile = blockIdx.x / team, tile_step = gridDim.x / team;
  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::kStages; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
    for (int s = 0; s < Cfg::kSfStages; ++s) {
      mbar_init(sf_full_bar(s), 1); mbar_init(sf_empty_bar(s), 1); mbar_init(sf_ready_bar(s), Cfg::kSfBlocks * (PAIR ? 2 : 1));
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full_bar(b), 1); mbar_init(acc_empty_bar(b), Cfg::kEpiWarps * (PAIR ? 2 : 1));
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tmap(&tmap_m); prefetch_tmap(&tmap_n); prefetch_tmap(&tmap_sm); prefetch_tmap(&tmap_sn);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(Cfg::kTmemCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(smem_u32(tmem_slot), Cfg::kTmemCols);
    }
    pdl_launch_dependents();
  }
  pdl_wait();                       // no global memory is touched before this
  if (warp == 2) {                  // the groups' first rows (clamped to what exists) and tiles
    const int col_tiles = static_cast<int>((p.n + kColsC - 1) / kColsC);
    int before = 0, reached = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
      const int g = g0 + lane;
      // rows start where the largest offset so far says: groups never overlap, whatever the offsets hold
      int first = 0, end = static_cast<int>(p.m);
      if (p.offsets) {
        auto offset = [&](int i) {
          const int o = p.offsets[i < p.groups ? i : p.groups];
          return o < 0 ? 0 : o > p.m ? static_cast<int>(p.m) : o;
        };
        first = offset(g);
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, first, s);
          if (lane >= s) first = max(first, up);
        }
        first = max(first, reached);
        end = max(first, offset(g + 1));
        reached = __shfl_sync(0xffffffffu, first, 31);
      }
      int tiles = 0;
      if (g < p.groups) {
        row_start[g] = first;
        if (g == p.groups - 1) row_start[p.groups] = end;
        tiles = ((end - first + kRows - 1) / kRows) * col_tiles;
      }
      int inc = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      if (g < p.groups) tile_start[g + 1] = before + inc;
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) tile_start[0] = 0;
  }
  tc_fence_before();
  __syncthreads();
  if (team > 1) cluster_sync_all();       // every CTA's barriers are initialised before anyone signals across
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int total_tiles = tile_start[p.groups];
  // this CTA's chunks of kChunk stages
  const int all_chunks = (p.k_blocks + kChunk - 1) / kChunk;
  const int per = PAIR ? all_chunks : (all_chunks + team - 1) / team;
  const int chunk0 = PAIR ? 0 : rank * per;
  const int chunk1 = min(all_chunks, chunk0 + per);
  const int kb0 = kChunk * chunk0, kb1 = min(p.k_blocks, kChunk * chunk1);       // its stages
  int group = 0;
  MxTile t;

  if (warp == 0) {
    // ---------------- TMA producer
    if (lane == 0) {
      int stage = 0, sf = 0;
      uint32_t phase = 0, sf_phase = 0, issued = 0;
      bool ok = true;
      for (int tile = first_tile; tile < total_tiles && ok; tile += tile_step) {
        find_tile<kRows, kColsC>(tile, tile_start, row_start, group, t);
        const int m0 = SWAP ? t.n0 : t.row0 + (PAIR ? rank * kTileM : 0);
        const int n0 = SWAP ? t.row0 : t.n0 + (PAIR ? rank * Cfg::kNRows : 0);
        const int zm = SWAP ? t.group : 0, zn = SWAP ? 0 : t.group;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (kb % kChunk == 0) {
            if (!mbar_wait(sf_empty_bar(sf), sf_phase ^ 1u, abort_flag, p.err)) { ok = false; break; }
            const uint32_t dst = base + Cfg::kSfOff + sf * Cfg::kSfStage;
            mbar_expect_tx(sf_full_bar(sf), (kTileM + BN) * 32);
            tma_load_3d(dst, &tmap_sm, kb * (kStageK / 32), m0, zm, sf_full_bar(sf));
            tma_load_3d(dst + kTileM * 32, &tmap_sn, kb * (kStageK / 32), SWAP ? t.row0 : t.n0, zn, sf_full_bar(sf));
            if (++sf == Cfg::kSfStages) { sf = 0; sf_phase ^= 1u; }
          }
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.err)) { ok = false; break; }
          const uint32_t dst = base + stage * Cfg::kStage;
          if constexpr (PAIR) {                       // both CTAs' bytes complete on the leader's barrier
            const uint32_t leader = map_to_cta(full_bar(stage), 0);
            if (rank == 0) mbar_expect_tx(full_bar(stage), 2 * Cfg::kStage);
            tma_load_3d_pair(dst, &tmap_m, kb * 128, m0, zm, leader);
            tma_load_3d_pair(dst + kTileM * 128, &tmap_n, kb * 128, n0, zn, leader);
            ++issued;
          } else {
            mbar_expect_tx(full_bar(stage), Cfg::kStage);
            tma_load_3d(dst, &tmap_m, kb * 128, m0, zm, full_bar(stage));
            tma_load_3d(dst + kTileM * 128, &tmap_n, kb * 128, n0, zn, full_bar(stage));
          }
          if (++stage == Cfg::kStages) { stage = 0; phase ^= 1u; }
        }
      }
      // whoever gives up, the loads land before the CTA leaves; a pair's codes, which land on the leader's barriers, at its end
      if constexpr (PAIR) store_cluster(map_to_cta(smem_u32(tmem_slot + 2 + rank), 0), issued);
      else ring_drain(Cfg::kStages, stage, phase, full_bar);
      ring_drain(Cfg::kSfStages, sf, sf_phase, sf_full_bar);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (the pair's leader only)
    if (!PAIR || rank == 0) {
      const uint32_t idesc0 = mx_idesc(BN, PAIR ? 256 : 128, 0), idesc2 = mx_idesc(BN, PAIR ? 256 : 128, 2);
      const uint32_t elected = elect_one();
      int stage = 0, sf = 0, acc = 0;
      uint32_t phase = 0, sf_phase = 0, acc_phase = 0;
      bool ok = true, here = false, sf_here = false;
      for (int tile = first_tile; tile < total_tiles && ok; tile += tile_step) {
        if (!warp_wait<PAIR>(acc_empty_bar(acc), acc_phase ^ 1u, abort_flag, p.err)) break;
        const uint32_t d = tmem + static_cast<uint32_t>(acc * BN);
        for (int kb = kb0; kb < kb1; ++kb) {
          const uint32_t part = static_cast<uint32_t>(kb) % kChunk;          // of the chunk
          // the next barriers were looked at while the last stage's instructions went out
          if (part == 0 && !sf_here && !warp_wait<PAIR>(sf_ready_bar(sf), sf_phase, abort_flag, p.err)) { ok = false; break; }
          if (!here && !warp_wait<PAIR>(full_bar(stage), phase, abort_flag, p.err)) { ok = false; break; }
          tc_fence_after();
          // the stage's codes have landed, so the instructions that used its columns of exponents before are done
          const uint32_t sfb = tmem + static_cast<uint32_t>(Cfg::kSfBase + stage * Cfg::kSfCols), sfa = sfb + 2 * Cfg::kSfN;
          const uint32_t sfs = base + Cfg::kSfOff + sf * Cfg::kSfStage + part * 1024;
          const uint32_t sm = desc_lo(base) + static_cast<uint32_t>(stage) * (Cfg::kStage >> 4), sn = sm + kTileM * 8;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            tmem_copy<MODE>(elected, sfa + w * 4, sfs + w * 512);
#pragma unroll
            for (int i = 1; i < Cfg::kSfBlocks; ++i) tmem_copy<MODE>(elected, sfb + w * Cfg::kSfN + (i - 1) * 4, sfs + i * 4096 + w * 512);
          }
          const bool sf_done = part == kChunk - 1 || kb + 1 == kb1;
          if (sf_done) commit_to<MODE>(elected, sf_empty_bar(sf));
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_mxf4<MODE>(elected, d, sm + kk * 2, sn + kk * 2, (kk & 1) ? idesc2 : idesc0, sfa + (kk >> 1) * 4, sfb + (kk >> 1) * Cfg::kSfN,
                           (kb > kb0 || kk > 0) ? 1u : 0u);
          commit_to<MODE>(elected, empty_bar(stage));
          if (kb + 1 == kb1) commit_to<MODE>(elected, acc_full_bar(acc));
          if (++stage == Cfg::kStages) { stage = 0; phase ^= 1u; }
          if (sf_done && ++sf == Cfg::kSfStages) { sf = 0; sf_phase ^= 1u; }
          here = __all_sync(0xffffffffu, mbar_test<PAIR>(full_bar(stage), phase));
          sf_here = sf_done && __all_sync(0xffffffffu, mbar_test<PAIR>(sf_ready_bar(sf), sf_phase));
        }
        if (++acc == Cfg::kAccs) { acc = 0; acc_phase ^= 1u; }
      }
      // and the instructions that were issued end before it gives its tensor memory back
      const int last = ring_last_slot(Cfg::kStages, stage);
      mbar_drain(empty_bar(last), ring_last_parity(last, stage, phase));
    }
  } else if (warp >= 2 + Cfg::kEpiWarps) {
    // ---------------- exponents: blocks of 128 rows, turned in place: row r's words w -> lane r % 32 of word w
    int sf = 0;
    uint32_t sf_phase = 0;
    bool ok = true;
    for (int tile = first_tile; tile < total_tiles && ok; tile += tile_step) {
      for (int c = chunk0; c < chunk1; ++c) {
        if (!warp_wait(sf_full_bar(sf), sf_phase, abort_flag, p.err)) { ok = false; break; }
        for (int block = warp - 2 - Cfg::kEpiWarps; block < Cfg::kSfBlocks; block += 2) {
          uint4 *rows = reinterpret_cast<uint4 *>(gen + Cfg::kSfOff + sf * Cfg::kSfStage + block * 4096);
          uint4 lo[4], hi[4];                          // rows lane, 32 + lane, ..: words 0-3 and 4-7
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            lo[j] = rows[2 * (32 * j + lane)];
            hi[j] = rows[2 * (32 * j + lane) + 1];
          }
          __syncwarp();
          rows[lane] = make_uint4(lo[0].x, lo[1].x, lo[2].x, lo[3].x);
          rows[32 + lane] = make_uint4(lo[0].y, lo[1].y, lo[2].y, lo[3].y);
          rows[64 + lane] = make_uint4(lo[0].z, lo[1].z, lo[2].z, lo[3].z);
          rows[96 + lane] = make_uint4(lo[0].w, lo[1].w, lo[2].w, lo[3].w);
          rows[128 + lane] = make_uint4(hi[0].x, hi[1].x, hi[2].x, hi[3].x);
          rows[160 + lane] = make_uint4(hi[0].y, hi[1].y, hi[2].y, hi[3].y);
          rows[192 + lane] = make_uint4(hi[0].z, hi[1].z, hi[2].z, hi[3].z);
          rows[224 + lane] = make_uint4(hi[0].w, hi[1].w, hi[2].w, hi[3].w);
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            if constexpr (PAIR) mbar_arrive_leader(map_to_cta(sf_ready_bar(sf), 0));
            else mbar_arrive(sf_ready_bar(sf));
          }
        }
        if (++sf == Cfg::kSfStages) { sf = 0; sf_phase ^= 1u; }
      }
    }
  } else {
    // ---------------- epilogue
    const int quad = warp & 3;
    uint8_t *stage = gen + Cfg::kEpiOff + (warp - 2) * (Cfg::kEpiBufs * 4096);
    const uint32_t stage_addr = base + Cfg::kEpiOff + (warp - 2) * (Cfg::kEpiBufs * 4096);
    constexpr int kCols = BN / (Cfg::kEpiWarps / 4);         // this warp's columns of a tile, from c_first on
    const int c_first = (warp - 2) / 4 * kCols;
    int acc = 0;
    uint32_t acc_phase = 0, nstores = 0;
    bool ok = true;
    for (int tile = first_tile; tile < total_tiles && ok; tile += tile_step) {
      find_tile<kRows, kColsC>(tile, tile_start, row_start, group, t);
      if constexpr (!SWAP && Cfg::kAccs == 1) {       // the tile's bias into the staging buffer, which is idle until then
        if (p.bias) {
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
          const int64_t n0 = t.n0 + c_first;
          for (int c = lane; c < kCols; c += 32)
            reinterpret_cast<float *>(stage)[c] = n0 + c < p.n ? load_float(p.bias, p.bias_dtype, t.group * p.bias_stride + n0 + c) : 0.0f;
          __syncwarp();
        }
      }
      bool landed = warp_wait(acc_full_bar(acc), acc_phase, abort_flag, p.err);
      if constexpr (SWAP) landed = epilogue_barrier(landed);        // all four warps go on or none; the tile before has left
      if (!landed) break;
      tc_fence_after();
      const uint32_t src = tmem + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(acc * BN);
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR) mbar_arrive_leader(map_to_cta(acc_empty_bar(acc), 0));
          else mbar_arrive(acc_empty_bar(acc));
        }
      };
      if constexpr (SWAP) {                           // lane = column of C, register = row
        if (team == 1) {                              // through shared memory: rows of C leave in 8- or 16-byte pieces
          uint8_t *tile_s = gen + Cfg::kEpiOff;
          store_partial_swapped<BN>(tile_s, src, quad * 32 + lane);
          release();
          epilogue_barrier(true);
          const int64_t col = t.n0 + 4 * lane;
          float bias[4];
          load_bias4(p, t.group, col, bias);
          const int rows = t.row_end - t.row0 < BN ? t.row_end - t.row0 : BN;
          for (int r0 = warp - 2; r0 < rows; r0 += 16) {
            float4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int row = r0 + 4 * u;             // inside the staging buffer: BN is a multiple of 16
              v[u] = *reinterpret_cast<const float4 *>(tile_s + row * (kTileM * 4) + ((lane ^ (row & 7)) * 16));
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (r0 + 4 * u < rows) store_piece(p, t.row0 + r0 + 4 * u, col, v[u], bias);
          }
        } else {                                      // joined below
          store_partial_swapped<BN>(gen, src, quad * 32 + lane);
        }
      } else {
        const int row0 = t.row0 + (PAIR ? rank * kTileM : 0) + quad * 32;
        if (MODE == kSingle && team > 1) {            // the partial tile into the ring, which is done with; joined below
          if (row0 < t.row_end) store_partial<BN>(gen, src, quad * 32 + lane);
        } else if (row0 < t.row_end) {
          RowWriter<Cfg::kEpiBufs> out(p, &tmap_out, t, row0, lane, stage, stage_addr, nstores);
          store_rows<kCols, Cfg::kAccs == 1>(p, out, src + static_cast<uint32_t>(c_first), t.group, t.n0 + c_first, lane, release);
        } else {
          release();
        }
      }
      if (++acc == Cfg::kAccs) { acc = 0; acc_phase ^= 1u; }
    }
    if (!SWAP && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  if constexpr (!PAIR) {
    if (team > 1) {                       // every CTA joins its share of the tile's rows
      __syncthreads();
      cluster_sync_all();
      group = 0;
      if (first_tile < total_tiles) {
        find_tile<kRows, kColsC>(first_tile, tile_start, row_start, group, t);
        if (team == 2) join_partials<kRows, Cfg::kThreads, 2>(p, t, base, rank);
        else if (team == 4) join_partials<kRows, Cfg::kThreads, 4>(p, t, base, rank);
        else join_partials<kRows, Cfg::kThreads, 8>(p, t, base, rank);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  // a peer may still signal into this CTA or read its shared memory
  if constexpr (PAIR) {
    uint32_t again = smem_u32(smem_raw);          // worked out anew: kept from above it costs the epilogue registers that it spills
    asm volatile("" : "+r"(again));
    again = ((again + 1023u) & ~1023u) + Cfg::kBarOff;
    pair_leave(again + 8 * (kB3 + 4) + 4, again, Cfg::kStages, Cfg::kStage);
  } else if (team > 1) {
    cluster_sync_all();
  }
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::kTmemCols) : "memory");
    else tmem_dealloc(tmem, Cfg::kTmemCols);
  }
}

struct MxOperand {
  const uint8_t *codes, *scales;
  int64_t code_stride, scale_stride, code_bs, scale_bs;   // bytes between rows and between matrices
  int64_t rows, batch;
};

// How many clusters of `split` CTAs run at once on the current device (a GPC's SMs are shared out in whole clusters, and
// which SMs it has differs from GPU to GPU).  Asked once per device.
template <int BN, int MODE> int64_t clusters_at_once(int split) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices][4];                     // the number + 1
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device >= kDevices) return 0;
  std::atomic<int> &slot = known[device][split == 2 ? 1 : split == 4 ? 2 : 3];
  int n = slot.load(std::memory_order_relaxed) - 1;
  if (n < 0) {
    using Cfg = MxCfg<BN, MODE>;
    cudaFuncSetAttribute(mxfp4_gemm_kernel<BN, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(split));
    cfg.blockDim = dim3(Cfg::kThreads);
    cfg.dynamicSmemBytes = Cfg::kSmem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(split);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, mxfp4_gemm_kernel<BN, MODE>, &cfg) != cudaSuccess) {
      cudaGetLastError();
      return 0;                    // not remembered: the next call asks again
    }
    slot.store(n + 1, std::memory_order_relaxed);
  }
  return n;
}

template <int BN, int MODE>
int32_t launch_mx(const MxOperand &a, const MxOperand &b, int64_t k, MxParams p, int split, int64_t max_tiles, cudaStream_t st) {
  using Cfg = MxCfg<BN, MODE>;
  const MxOperand &om = MODE == kFew ? b : a, &on = MODE == kFew ? a : b;
  CUtensorMap tm, tn, tsm, tsn, tout{};
  const uint64_t kb = static_cast<uint64_t>((k + 1) / 2), ks = static_cast<uint64_t>(ceil_div(k, 32));
  const int eb = dtype_bytes(p.out_dtype);
  if (!make_byte_tmap3(&tm, om.codes, kb, om.rows, om.batch, om.code_stride, om.code_bs, 128, kTileM, true) ||
      !make_byte_tmap3(&tn, on.codes, kb, on.rows, on.batch, on.code_stride, on.code_bs, 128, Cfg::kNRows, true) ||
      !make_byte_tmap3(&tsm, om.scales, ks, om.rows, om.batch, om.scale_stride, om.scale_bs, 32, kTileM, false) ||
      !make_byte_tmap3(&tsn, on.scales, ks, on.rows, on.batch, on.scale_stride, on.scale_bs, 32, BN, false) ||
      (MODE != kFew && p.tma_out && !make_byte_tmap(&tout, p.out, p.n * eb, p.m, p.ldo * eb, 32)))
    return fail(BSIR_ERR_STRIDE, "matmul_mxfp4: the driver refuses a tensor map of these sizes and strides");
  cudaFuncSetAttribute(mxfp4_gemm_kernel<BN, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
  const int team = MODE == kPair ? 2 : split;
  p.split = team;
  int64_t teams = (device_info().sm_count > 0 ? device_info().sm_count : 148) / team;
  if (teams > max_tiles || (MODE != kPair && split > 1)) teams = max_tiles;     // a cluster that shares K has one tile
  const dim3 grid(static_cast<unsigned>(teams * team));
  if (team > 1) launch_pdl_cluster(mxfp4_gemm_kernel<BN, MODE>, grid, dim3(Cfg::kThreads), Cfg::kSmem, st, team, tm, tn, tsm, tsn, tout, p);
  else launch_pdl(mxfp4_gemm_kernel<BN, MODE>, grid, dim3(Cfg::kThreads), Cfg::kSmem, st, tm, tn, tsm, tsn, tout, p);
  count_launch();
  return check_launch("matmul_mxfp4");
}

struct MxForm {
  MxMode mode;
  int rows, cols;        // of C in a tile
  int split;             // CTAs that work on one
  int64_t tiles;         // at most
};
MxForm choose_form(int64_t m, int64_t n, int64_t k, int64_t groups) {
  // Which form: from the rows of a group, all of them or one and a half times the groups' mean, which most groups stay
  // under (their sizes are on the device; a group that needs a second tile reads its weights twice.  128 groups of 16 rows
  // on average, 4096 x 1536: 90 us in tiles of 16, 74 in tiles of 32; of 32 rows: 93 in tiles of 32, 78 in tiles of 64).
  const int64_t rows = groups > 1 ? ceil_div(3 * m, 2 * groups) : m, stages = ceil_div(k, kStageK), chunks = ceil_div(stages, kChunk);
  const int64_t sms = device_info().sm_count > 0 ? device_info().sm_count : 148;
  auto tiles = [&](int64_t r, int64_t c) { return (groups > 1 ? m / r + groups : ceil_div(m, r)) * ceil_div(n, c); };   // at most
  // K may be shared out over a cluster if every CTA gets a part and all clusters are at work at once (37 of four CTAs in
  // two rounds: 13 us where one CTA a tile takes 8).
  auto can_split = [&](auto at_once, int64_t nt, int s) { return nt * s <= sms && ceil_div(chunks, s) * (s - 1) < chunks && nt <= at_once(s); };
  if (rows <= 32) {
    // the more CTAs the better (1 row, N x K = 4096 x 4096: 6.7 us whole, 6.4 by two, 6.2 by four; 4096 x 14336: 15.4,
    // 11.2, 9.6); kSingle takes 8.2 and 18 to 21 us there, and 10 to 13 us on 14336 x 4096, where this takes 8.7 to 9.9
    int split = 1;
    auto widest = [&](auto at_once, int64_t nt) {
      for (int s = 8; s > 1 && split == 1; s /= 2)
        if (can_split(at_once, nt, s)) split = s;
      return nt;
    };
    const int64_t nt = rows <= 16 ? widest(clusters_at_once<16, kFew>, tiles(16, kTileM)) : widest(clusters_at_once<32, kFew>, tiles(32, kTileM));
    return {kFew, rows <= 16 ? 16 : 32, kTileM, split, nt};
  }
  // Otherwise the least of these estimates, in units of 5 ns beside what every launch takes: rounds of tiles over the SMs x
  // (stages x a stage's time + a tile's own), plus the join of a shared K, which grows with the rows of a tile.  Measured
  // over 33 .. 4096 rows, N x K from 1000 x 8192 to 40000 x 1024.  Groups leave half of a last tile empty on average, and
  // their last round is half full.
  auto cost = [&](int64_t r, int64_t c, int64_t at_once, int64_t tile) {
    if (groups == 1) return ceil_div(tiles(r, c), at_once) * tile;
    const int64_t most = m < groups ? m : groups, mean = m / r + groups / 2 + 1;     // every group has a tile
    return (mean < most ? most : mean) * ceil_div(n, c) * tile / at_once + tile / 2;
  };
  auto part = [&](int s) { return kChunk * ceil_div(chunks, s); };            // stages of a CTA
  const int64_t r64 = rows < 64 ? rows : 64, r128 = rows < 128 ? rows : 128;
  const int64_t tail = groups > 1 ? 128 : 0;              // rows next to another group's are stored by the warps
  int64_t few = cost(64, kTileM, sms, 50 * stages + 5 * (r64 - 24)), single = cost(kTileM, 128, sms, 61 * stages + tail);
  int few_split = 1, single_split = 1;
  for (int s = 2; s <= 8; s *= 2) {
    const int64_t f = s == 2 ? 51 * part(s) + 180 + 23 * r64 / 10 : 58 * part(s) + (s == 4 ? 370 : 470) + 24 * r64 / 10;
    if (f < few && can_split(clusters_at_once<64, kFew>, tiles(64, kTileM), s)) { few = f; few_split = s; }
    const int64_t g = s == 2 ? 57 * part(s) + 240 + 26 * r128 / 10 : 63 * part(s) + (s == 4 ? 350 : 450) + 41 * r128 / 10;
    if (g < single && can_split(clusters_at_once<128, kSingle>, tiles(kTileM, 128), s)) { single = g; single_split = s; }
  }
  const int64_t pair = cost(256, 256, sms / 2, 69 * stages + 260 + tail);
  if (few < single && few < pair) return {kFew, 64, kTileM, few_split, tiles(64, kTileM)};
  if (single <= pair) return {kSingle, kTileM, 128, single_split, tiles(kTileM, 128)};
  return {kPair, 256, 256, 2, tiles(256, 256)};
}

}  // namespace
}  // namespace bsir

using namespace bsir;

extern "C" int32_t bsir_matmul_mxfp4_form(int64_t m, int64_t n, int64_t k, int64_t groups, int32_t *tile_rows, int32_t *tile_cols, int32_t *tile_ctas) {
  clear_error();
  constexpr int64_t kMax = int64_t{1} << 30;
  if (m < 1 || n < 1 || k < 1 || m > kMax || n > kMax || k > kMax || m > (int64_t{1} << 40) / n || groups < 1 || groups > kMaxGroups)
    return fail(BSIR_ERR_SHAPE, "matmul_mxfp4_form: m %lld, n %lld, k %lld (1 to 2^30, at most 2^40 results), %lld groups (1 to %d)", (long long)m,
                (long long)n, (long long)k, (long long)groups, kMaxGroups);
  if (!tile_rows || !tile_cols || !tile_ctas) return fail(BSIR_ERR_NULL, "matmul_mxfp4_form: null pointer");
  const MxForm f = choose_form(m, n, k, groups);
  *tile_rows = f.rows; *tile_cols = f.cols; *tile_ctas = f.split;
  return BSIR_OK;
}

extern "C" int32_t bsir_matmul_mxfp4(const bsir_matmul_mxfp4_desc *d, void *stream) {
  clear_error();
  if (!d) return fail(BSIR_ERR_NULL, "matmul_mxfp4: null description");
  if (!dtype_is_float(d->out_dtype)) return fail(BSIR_ERR_DTYPE, "matmul_mxfp4: out dtype %d (f32, f16, bf16)", d->out_dtype);
  if (d->bias && !dtype_is_float(d->bias_dtype)) return fail(BSIR_ERR_DTYPE, "matmul_mxfp4: bias dtype %d (f32, f16, bf16)", d->bias_dtype);
  constexpr int64_t kMax = int64_t{1} << 30;
  if (d->m < 0 || d->n < 0 || d->k < 1 || d->m > kMax || d->n > kMax || d->k > kMax)
    return fail(BSIR_ERR_SHAPE, "matmul_mxfp4: m %lld, n %lld, k %lld (k at least 1, none above 2^30)", (long long)d->m, (long long)d->n, (long long)d->k);
  if (d->offsets ? (d->groups < 1 || d->groups > kMaxGroups) : d->groups > 1)
    return fail(BSIR_ERR_SHAPE, "matmul_mxfp4: %lld groups (1 to %d with offsets, at most 1 without)", (long long)d->groups, kMaxGroups);
  if (d->m == 0 || d->n == 0) return BSIR_OK;
  if (!d->a || !d->scale_a || !d->b || !d->scale_b || !d->out) return fail(BSIR_ERR_NULL, "matmul_mxfp4: null pointer");
  const int64_t groups = d->offsets ? d->groups : 1;
  const int64_t kb = (d->k + 1) / 2, ks = ceil_div(d->k, 32);
  const int64_t kb16 = ceil_div(kb, 16) * 16, ks16 = ceil_div(ks, 16) * 16;
  MxOperand a{d->a, d->scale_a, d->lda, d->ldsa, 0, 0, d->m, 1}, b{d->b, d->scale_b, d->ldb, d->ldsb, d->batch_stride_b, d->batch_stride_sb, d->n, groups};
  for (MxOperand *o : {&a, &b}) {
    const char *name = o == &a ? "a" : "b";
    if (o->rows == 1) { o->code_stride = kb16; o->scale_stride = ks16; }      // a lone row's pitch means nothing
    if (o->batch == 1) { o->code_bs = o->rows * o->code_stride; o->scale_bs = o->rows * o->scale_stride; }
    if (o->code_stride < kb || o->scale_stride < ks || o->code_stride % 16 || o->scale_stride % 16)
      return fail(BSIR_ERR_STRIDE, "matmul_mxfp4: row strides of %s: codes %lld bytes (at least %lld), exponents %lld (at least %lld), multiples of 16", name,
                  (long long)o->code_stride, (long long)kb, (long long)o->scale_stride, (long long)ks);
    if (o->code_bs % 16 || o->scale_bs % 16 || o->code_bs < (o->rows - 1) * o->code_stride + kb || o->scale_bs < (o->rows - 1) * o->scale_stride + ks)
      return fail(BSIR_ERR_STRIDE, "matmul_mxfp4: group strides of %s: codes %lld bytes, exponents %lld: multiples of 16 that hold a matrix", name,
                  (long long)o->code_bs, (long long)o->scale_bs);
    if (!aligned_to(o->codes, 16) || !aligned_to(o->scales, 16)) return fail(BSIR_ERR_ALIGN, "matmul_mxfp4: %s and its exponents want 16-byte aligned bases", name);
  }
  if (d->bias && d->bias_stride < 0) return fail(BSIR_ERR_STRIDE, "matmul_mxfp4: %lld elements between the groups' biases", (long long)d->bias_stride);
  const int eb = dtype_bytes(d->out_dtype);
  const int64_t ldo = d->m == 1 ? d->n : d->ldo;
  if (ldo < d->n) return fail(BSIR_ERR_STRIDE, "matmul_mxfp4: row stride %lld of out for %lld columns", (long long)ldo, (long long)d->n);
  if (!aligned_to(d->out, eb) || (d->offsets && !aligned_to(d->offsets, 4)) || (d->bias && !aligned_to(d->bias, dtype_bytes(d->bias_dtype))))
    return fail(BSIR_ERR_ALIGN, "matmul_mxfp4: out, offsets or bias misaligned");
  {
    const char *o0 = static_cast<const char *>(d->out), *o1 = o0 + ((d->m - 1) * ldo + d->n) * eb;
    const int64_t nbias = d->bias ? ((groups - 1) * d->bias_stride + d->n) * dtype_bytes(d->bias_dtype) : 0;
    struct { const void *p; int64_t bytes; } in[6] = {
        {a.codes, (a.rows - 1) * a.code_stride + kb}, {a.scales, (a.rows - 1) * a.scale_stride + ks},
        {b.codes, (groups - 1) * b.code_bs + (b.rows - 1) * b.code_stride + kb}, {b.scales, (groups - 1) * b.scale_bs + (b.rows - 1) * b.scale_stride + ks},
        {d->bias, nbias}, {d->offsets, d->offsets ? (groups + 1) * 4 : 0}};
    for (const auto &i : in) {
      const char *i0 = static_cast<const char *>(i.p);
      if (i.bytes > 0 && i0 < o1 && o0 < i0 + i.bytes) return fail(BSIR_ERR_UNSUPPORTED, "matmul_mxfp4: out may not overlap an operand");
    }
  }
  MxParams p{};
  p.m = d->m; p.n = d->n; p.k_blocks = static_cast<int>(ceil_div(d->k, kStageK));
  p.offsets = d->offsets; p.groups = static_cast<int>(groups);
  p.bias = d->bias; p.bias_stride = d->bias_stride; p.bias_dtype = d->bias_dtype; p.out_dtype = d->out_dtype;
  p.out = d->out; p.ldo = ldo;
  p.err = device_error_word();
  if (!p.err) return fail(BSIR_ERR_WORKSPACE, "matmul_mxfp4: no device error word");
  cudaStream_t st = resolve_stream(stream);
  p.tma_out = aligned_to(d->out, 16) && (ldo * eb) % 16 == 0 && d->n * eb <= 0x7fffffff;     // its coordinates are 32-bit bytes
  const MxForm f = choose_form(d->m, d->n, d->k, groups);
  if (f.mode == kPair) return launch_mx<256, kPair>(a, b, d->k, p, 1, f.tiles, st);
  if (f.mode == kSingle) return launch_mx<128, kSingle>(a, b, d->k, p, f.split, f.tiles, st);
  if (f.rows == 64) return launch_mx<64, kFew>(a, b, d->k, p, f.split, f.tiles, st);
  if (f.rows == 32) return launch_mx<32, kFew>(a, b, d->k, p, f.split, f.tiles, st);
  return launch_mx<16, kFew>(a, b, d->k, p, f.split, f.tiles, st);
}
