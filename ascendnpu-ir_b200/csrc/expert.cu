// expert.cu -- a mixture-of-experts layer's bookkeeping and data movement: tokens sorted by expert and back.
//
//   ids[t, j]      the expert of token t's j-th choice; a number outside [0, experts) names none ("masked")
//   offsets[e]     first row of expert e; offsets[experts] = the number of rows
//   slots[t, j]    the row of choice (t, j), -1 for a masked one.  Rows of one expert keep the order of (t, j).
//   dispatch       rows[slots[t, j]] = x[t]
//   combine        out[t] = sum_j w[t, j] * y[slots[t, j]]               (w = 1 without weights: dispatch's gradient)
//   its gradient   dy[slots[t, j]] = w[t, j] * dout[t],   dw[t, j] = <dout[t], y[slots[t, j]]>
//
// Everything goes by token, not by row: a token's row is read once and its copies leave from registers (by row, each
// copy's source would be fetched again, as the rows of one token lie far apart), and a token's sum is made in j order
// by one thread per column, so no atomics and the same bits on every run.  Masked choices touch nothing: no row of y
// is read for them, rows that no choice names keep their contents.  Slots come from device memory, so the kernels check
// them: one that is neither -1 nor a row is treated as masked and raises BSIR_DEVERR_GATHER_INDEX.
#include "common.cuh"

namespace bsir {
namespace {

// ------------------------------------------------------------------------------------------------ sort
// A stable counting sort.  A CTA counts the experts of its 4096 choices per warp (each warp owns 128 consecutive
// choices, 32 at a time: the lanes with one expert find each other with match.any, and a choice's rank among them is a
// popcount), and the counts of the warps before it, of the CTAs before it and of the experts before its own add up to a
// choice's row.  Up to 4096 choices are one CTA and one launch; more take a counting launch first, whose table of
// [experts] counts per CTA the placing launch adds up.
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortPerWarp = 128;
constexpr int kSortChunk = kSortWarps * kSortPerWarp;
constexpr int kMaxExperts = 1024;

struct SortParams {
  const void *ids;
  int64_t n;                  // choices
  int experts;
  int wide;                   // ids are int64
  int32_t *offsets, *slots;
  int32_t *table;             // [chunks][experts] counts, null with one chunk
  int chunks;
};
__device__ __forceinline__ int load_id(const SortParams &p, int64_t i) {
  if (i >= p.n) return -1;
  if (p.wide) {
    const long long v = static_cast<const long long *>(p.ids)[i];
    return v >= 0 && v < p.experts ? static_cast<int>(v) : -1;
  }
  const int v = static_cast<const int *>(p.ids)[i];
  return v >= 0 && v < p.experts ? v : -1;
}

// exclusive prefix sum over `count[0 .. experts)` by the whole CTA (experts <= kSortThreads); returns this thread's
// prefix, *total the sum
__device__ __forceinline__ int cta_prefix(int v, int *warp_sum_s, int *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) warp_sum_s[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sum_s[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += up;
    }
    warp_sum_s[lane] = s;
  }
  __syncthreads();
  *total = warp_sum_s[kSortWarps - 1];
  return inc - v + (warp ? warp_sum_s[warp - 1] : 0);
}

__global__ void __launch_bounds__(kSortThreads) expert_count_kernel(SortParams p) {
  __shared__ int count[kMaxExperts];
  for (int e = threadIdx.x; e < p.experts; e += kSortThreads) count[e] = 0;
  pdl_launch_dependents();
  pdl_wait();
  __syncthreads();
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) * kSortChunk;
#pragma unroll
  for (int u = 0; u < kSortChunk / kSortThreads; ++u) {
    const int id = load_id(p, c0 + u * kSortThreads + threadIdx.x);
    if (id >= 0) atomicAdd(&count[id], 1);       // integers: the order does not show
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += kSortThreads) p.table[static_cast<int64_t>(blockIdx.x) * p.experts + e] = count[e];
}

__global__ void __launch_bounds__(kSortThreads) expert_place_kernel(SortParams p) {
  extern __shared__ uint16_t warp_count[];       // [experts][kSortWarps]: choices of an expert per warp, then before a warp
  __shared__ int base_s[kMaxExperts];
  __shared__ int warp_sum_s[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < p.experts * kSortWarps / 2; i += kSortThreads) reinterpret_cast<uint32_t *>(warp_count)[i] = 0;
  pdl_launch_dependents();
  pdl_wait();
  __syncthreads();
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) * kSortChunk + warp * kSortPerWarp;
  int id[kSortPerWarp / 32], rank[kSortPerWarp / 32];
#pragma unroll
  for (int u = 0; u < kSortPerWarp / 32; ++u) id[u] = load_id(p, c0 + u * 32 + lane);
#pragma unroll
  for (int u = 0; u < kSortPerWarp / 32; ++u) {
    const unsigned peers = __match_any_sync(0xffffffffu, id[u]);
    const int before = __popc(peers & ((1u << lane) - 1u));
    rank[u] = 0;
    if (id[u] >= 0) rank[u] = warp_count[id[u] * kSortWarps + warp] + before;   // 0 at first, then what the groups before left
    __syncwarp();
    if (id[u] >= 0 && before == 0) warp_count[id[u] * kSortWarps + warp] += static_cast<uint16_t>(__popc(peers));
    __syncwarp();
  }
  __syncthreads();
  // per expert: counts of the warps -> counts of the warps before, this chunk's total; of the other chunks: those before
  // this one and all
  int mine = 0, earlier = 0, all = 0;
  if (tid < p.experts) {
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = warp_count[tid * kSortWarps + w];
      warp_count[tid * kSortWarps + w] = static_cast<uint16_t>(mine);
      mine += c;
    }
    if (p.table) {
      for (int b = 0; b < p.chunks; ++b) {
        const int c = p.table[static_cast<int64_t>(b) * p.experts + tid];
        if (b < static_cast<int>(blockIdx.x)) earlier += c;
        all += c;
      }
    } else {
      all = mine;
    }
  }
  int total;
  const int start = cta_prefix(all, warp_sum_s, &total);
  if (tid < p.experts) {
    base_s[tid] = start + earlier;
    if (blockIdx.x == 0) p.offsets[tid] = start;
  }
  if (blockIdx.x == 0 && tid == 0) p.offsets[p.experts] = total;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kSortPerWarp / 32; ++u) {
    const int64_t i = c0 + u * 32 + lane;
    if (i < p.n) p.slots[i] = id[u] < 0 ? -1 : base_s[id[u]] + warp_count[id[u] * kSortWarps + warp] + rank[u];
  }
}

// ------------------------------------------------------------------------------------------------ movement
struct RowParams {
  int64_t tokens;
  int top_k;
  int64_t cols;               // elements of a row (dispatch: pieces of the copying type)
  int64_t rows;               // rows that slots may name
  const void *x;              // by token: dispatch's source, the gradient's dout
  int64_t xs;
  const void *y;              // by row
  int64_t ys;
  const int32_t *slots;
  const void *w;              // [tokens, top_k] or null
  int32_t w_dtype;
  void *out;                  // dispatch: by row; combine: by token
  int64_t os;
  void *dy;                   // by row
  int64_t dys;
  float *dw;
  int *err;
};
// The choices of a token, 32 at a time: lane j holds the slot (-1: masked; so is a number that names no row, which is
// reported) and the weight of choice j0 + j, loaded before the rows they lead to and handed round by shuffles.
struct Choices {
  int32_t slot;
  float weight;
  __device__ __forceinline__ void load(const RowParams &p, int64_t t, int j0) {
    const int lane = threadIdx.x & 31;
    slot = -1;
    weight = 1.0f;
    if (j0 + lane >= p.top_k) return;
    const int64_t i = t * p.top_k + j0 + lane;
    const int32_t s = p.slots[i];
    if (s >= 0 && s < p.rows) {
      slot = s;
      if (p.w) {
        if (p.w_dtype == BSIR_F32) {
          weight = static_cast<const float *>(p.w)[i];
        } else {
          const unsigned short h = static_cast<const unsigned short *>(p.w)[i];
          weight = p.w_dtype == BSIR_F16 ? __half2float(__ushort_as_half(h)) : __uint_as_float(static_cast<uint32_t>(h) << 16);
        }
      }
    } else if (s != -1) {
      atomicOr(p.err, BSIR_DEVERR_GATHER_INDEX);
    }
  }
  __device__ __forceinline__ int32_t slot_of(int j) const { return __shfl_sync(0xffffffffu, slot, j); }
  __device__ __forceinline__ float weight_of(int j) const { return __shfl_sync(0xffffffffu, weight, j); }
};

// Rows as pieces of type T (16 bytes where everything is aligned to it): a thread holds four pieces of the token's row
// and stores them to each of its rows.
constexpr int kMoveThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kMoveThreads) expert_dispatch_kernel(RowParams p) {
  pdl_launch_dependents();
  pdl_wait();
  for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    const T *src = static_cast<const T *>(p.x) + t * p.xs;
    Choices ch;
    ch.load(p, t, 0);
    for (int64_t c0 = static_cast<int64_t>(blockIdx.y) * (kMoveThreads * 4); c0 < p.cols; c0 += static_cast<int64_t>(gridDim.y) * (kMoveThreads * 4)) {
      T v[4];
      const int64_t c = c0 + threadIdx.x;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c + u * kMoveThreads < p.cols) v[u] = src[c + u * kMoveThreads];
      for (int j = 0; j < p.top_k; ++j) {
        if (p.top_k > 32 && j % 32 == 0) ch.load(p, t, j);
        const int64_t s = ch.slot_of(j % 32);
        if (s < 0) continue;
        T *dst = static_cast<T *>(p.out) + s * p.os;
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (c + u * kMoveThreads < p.cols) dst[c + u * kMoveThreads] = v[u];
      }
    }
  }
}

// A thread takes kE elements (16 bytes when kE > 1) of a token's row and runs over its choices, eight of y's rows in
// flight at a time.
template <int DT, bool VEC> struct RowVec {
  static constexpr int kPer = FloatTraits<DT>::kPerWord;
  static constexpr int kE = VEC ? 4 * kPer : 1;
  static constexpr int kW = VEC ? 4 : 1;
  uint32_t w[kW];
  __device__ __forceinline__ void load(const void *base, int64_t at) {
    if constexpr (VEC) {
      const Vec16 b = ld_stream(static_cast<const char *>(base) + at * (4 / kPer));
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = b.w[i];
    } else if constexpr (DT == BSIR_F32) {
      w[0] = static_cast<const uint32_t *>(base)[at];
    } else {
      w[0] = static_cast<const unsigned short *>(base)[at];
    }
  }
  __device__ __forceinline__ void get(float *v) const {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < 4; ++i) FloatTraits<DT>::unpack(w[i], v + i * kPer);
    } else {
      float t[2];
      FloatTraits<DT>::unpack(w[0], t);
      v[0] = t[0];
    }
  }
  __device__ static __forceinline__ void store(void *base, int64_t at, const float *v) {
    if constexpr (VEC) {
      Vec16 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o.w[i] = FloatTraits<DT>::pack(v + i * kPer);
      *reinterpret_cast<uint4 *>(static_cast<char *>(base) + at * (4 / kPer)) = make_uint4(o.w[0], o.w[1], o.w[2], o.w[3]);
    } else {
      const float t[2] = {v[0], 0.0f};
      const uint32_t w = FloatTraits<DT>::pack(t);
      if constexpr (DT == BSIR_F32) static_cast<uint32_t *>(base)[at] = w;
      else static_cast<unsigned short *>(base)[at] = static_cast<unsigned short>(w);
    }
  }
};

template <int DT, bool VEC>
__global__ void __launch_bounds__(kMoveThreads) expert_combine_kernel(RowParams p) {
  using V = RowVec<DT, VEC>;
  constexpr int kE = V::kE;
  pdl_launch_dependents();
  pdl_wait();
  for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    Choices ch;
    ch.load(p, t, 0);
    // the warp stays together for the shuffles: lanes behind the row's end go along without loading
    for (int64_t c0 = static_cast<int64_t>(blockIdx.y) * kMoveThreads * kE; c0 < p.cols; c0 += static_cast<int64_t>(gridDim.y) * kMoveThreads * kE) {
      const int64_t c = c0 + threadIdx.x * kE;
      const bool in = c < p.cols;
      float acc[kE];
#pragma unroll
      for (int i = 0; i < kE; ++i) acc[i] = 0.0f;
      for (int j0 = 0; j0 < p.top_k; j0 += 8) {
        if (p.top_k > 32 && j0 % 32 == 0) ch.load(p, t, j0);
        V v[8];
        uint32_t live = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int64_t s = ch.slot_of((j0 + u) % 32);      // lanes behind the last choice hold -1
          if (s >= 0) {
            live |= 1u << u;
            if (in) v[u].load(p.y, s * p.ys + c);
          }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float w = ch.weight_of((j0 + u) % 32);
          if (!(live >> u & 1u) || !in) continue;
          float f[kE];
          v[u].get(f);
#pragma unroll
          for (int i = 0; i < kE; ++i) acc[i] = __fmaf_rn(w, f[i], acc[i]);
        }
      }
      if (in) V::store(p.out, t * p.os + c, acc);
    }
  }
}

// One CTA per token, four choices at a time (eight took 120 registers and 267 us where four take 190): y's rows are
// read once, dy's written once, dout's once for the four; the dot products meet across the warps in a fixed order.
constexpr int kGradThreads = 128;
constexpr int kGradChoices = 4;
template <int DT, bool VEC>
__global__ void __launch_bounds__(kGradThreads) expert_combine_grad_kernel(RowParams p) {
  using V = RowVec<DT, VEC>;
  constexpr int kE = V::kE;
  __shared__ float part[kGradChoices][kGradThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    Choices ch;
    for (int j0 = 0; j0 < p.top_k; j0 += kGradChoices) {
      if (j0 % 32 == 0) ch.load(p, t, j0);
      int32_t s[kGradChoices];
      float w[kGradChoices], dot[kGradChoices];
#pragma unroll
      for (int u = 0; u < kGradChoices; ++u) {
        s[u] = ch.slot_of((j0 + u) % 32);
        w[u] = ch.weight_of((j0 + u) % 32);
        dot[u] = 0.0f;
      }
      for (int64_t c = static_cast<int64_t>(threadIdx.x) * kE; c < p.cols; c += static_cast<int64_t>(kGradThreads) * kE) {
        V g, y[kGradChoices];
        g.load(p.x, t * p.xs + c);
#pragma unroll
        for (int u = 0; u < kGradChoices; ++u)
          if (s[u] >= 0) y[u].load(p.y, s[u] * p.ys + c);
        float gf[kE];
        g.get(gf);
#pragma unroll
        for (int u = 0; u < kGradChoices; ++u) {
          if (s[u] < 0) continue;
          float yf[kE], o[kE];
          y[u].get(yf);
#pragma unroll
          for (int i = 0; i < kE; ++i) {
            dot[u] = __fmaf_rn(gf[i], yf[i], dot[u]);
            o[i] = __fmul_rn(w[u], gf[i]);
          }
          V::store(p.dy, s[u] * p.dys + c, o);
        }
      }
#pragma unroll
      for (int u = 0; u < kGradChoices; ++u) {
        dot[u] = warp_sum(dot[u]);
        if (lane == 0) part[u][warp] = dot[u];
      }
      __syncthreads();
      if (threadIdx.x < kGradChoices && j0 + static_cast<int>(threadIdx.x) < p.top_k) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kGradThreads / 32; ++i) sum += part[threadIdx.x][i];
        p.dw[t * p.top_k + j0 + threadIdx.x] = sum;       // 0 for a masked choice
      }
      __syncthreads();
    }
  }
}

int32_t check_choice(const char *what, int64_t tokens, int64_t top_k, int64_t cols, int64_t rows) {
  if (tokens < 0 || top_k < 0 || cols < 0 || rows < 0 || top_k > 0x7fffffff)
    return fail(BSIR_ERR_SHAPE, "%s: %lld tokens x %lld choices, %lld columns, %lld rows", what, (long long)tokens, (long long)top_k, (long long)cols,
                (long long)rows);
  if (top_k > 0 && tokens > 0x7fffffff / top_k)
    return fail(BSIR_ERR_SHAPE, "%s: %lld x %lld choices (at most 2^31 - 1)", what, (long long)tokens, (long long)top_k);
  return BSIR_OK;
}
int32_t check_stride(const char *what, const char *name, int64_t rows, int64_t cols, int64_t *stride) {
  if (rows <= 1) *stride = cols;      // a lone row's pitch means nothing
  if (*stride < cols) return fail(BSIR_ERR_STRIDE, "%s: row stride %lld of %s for %lld columns", what, (long long)*stride, name, (long long)cols);
  return BSIR_OK;
}
bool overlap(const void *a, int64_t na, const void *b, int64_t nb) {
  const char *a0 = static_cast<const char *>(a), *b0 = static_cast<const char *>(b);
  return na > 0 && nb > 0 && a0 < b0 + nb && b0 < a0 + na;
}
int64_t span(int64_t rows, int64_t cols, int64_t stride, int eb) { return rows > 0 ? ((rows - 1) * stride + cols) * eb : 0; }
bool rows_aligned(const void *p, int64_t stride, int eb) { return aligned_to(p, 16) && (stride * eb) % 16 == 0; }

// tokens along x; a row is cut along y when there are too few tokens to fill the SMs
dim3 move_grid(int64_t tokens, int64_t pieces_per_row) {
  const int sms = device_info().sm_count > 0 ? device_info().sm_count : 148;
  const int64_t gx = tokens < (int64_t{1} << 30) ? tokens : int64_t{1} << 30;
  int64_t gy = ceil_div(4 * sms, gx);
  if (gy > pieces_per_row) gy = pieces_per_row;
  return dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy < 1 ? 1 : (gy > 65535 ? 65535 : gy)));
}

template <int DT>
int32_t launch_combine(const RowParams &p, bool vec, cudaStream_t st) {
  if (vec) {
    launch_pdl(expert_combine_kernel<DT, true>, move_grid(p.tokens, ceil_div(p.cols, kMoveThreads * RowVec<DT, true>::kE)), dim3(kMoveThreads), 0, st, p);
  } else {
    launch_pdl(expert_combine_kernel<DT, false>, move_grid(p.tokens, ceil_div(p.cols, kMoveThreads)), dim3(kMoveThreads), 0, st, p);
  }
  count_launch();
  return check_launch("expert_combine");
}
template <int DT>
int32_t launch_combine_grad(const RowParams &p, bool vec, cudaStream_t st) {
  const unsigned grid = static_cast<unsigned>(p.tokens < (int64_t{1} << 30) ? p.tokens : int64_t{1} << 30);
  if (vec) launch_pdl(expert_combine_grad_kernel<DT, true>, dim3(grid), dim3(kGradThreads), 0, st, p);
  else launch_pdl(expert_combine_grad_kernel<DT, false>, dim3(grid), dim3(kGradThreads), 0, st, p);
  count_launch();
  return check_launch("expert_combine_grad");
}

}  // namespace
}  // namespace bsir

using namespace bsir;

extern "C" {

int32_t bsir_expert_sort(int32_t id_dtype, int64_t tokens, int64_t top_k, int64_t experts, const void *ids, int32_t *offsets, int32_t *slots,
                         void *stream) {
  clear_error();
  if (id_dtype != BSIR_I32 && id_dtype != BSIR_I64) return fail(BSIR_ERR_DTYPE, "expert_sort: id dtype %d (i32, i64)", id_dtype);
  if (int32_t rc = check_choice("expert_sort", tokens, top_k, 0, 0)) return rc;
  if (experts < 1 || experts > kMaxExperts) return fail(BSIR_ERR_SHAPE, "expert_sort: %lld experts (1 to %d)", (long long)experts, kMaxExperts);
  const int64_t n = tokens * top_k;
  if (!offsets || (n > 0 && (!ids || !slots))) return fail(BSIR_ERR_NULL, "expert_sort: null pointer");
  if (!aligned_to(ids, id_dtype == BSIR_I64 ? 8 : 4) || !aligned_to(offsets, 4) || !aligned_to(slots, 4)) return fail(BSIR_ERR_ALIGN, "expert_sort: misaligned");
  const int64_t id_bytes = n * (id_dtype == BSIR_I64 ? 8 : 4);
  if (overlap(ids, id_bytes, slots, n * 4) || overlap(ids, id_bytes, offsets, (experts + 1) * 4) || overlap(slots, n * 4, offsets, (experts + 1) * 4))
    return fail(BSIR_ERR_UNSUPPORTED, "expert_sort: ids, offsets and slots may not overlap");
  cudaStream_t st = resolve_stream(stream);
  SortParams p{};
  p.ids = ids; p.n = n; p.experts = static_cast<int>(experts); p.wide = id_dtype == BSIR_I64;
  p.offsets = offsets; p.slots = slots;
  p.chunks = static_cast<int>(n > 0 ? ceil_div(n, kSortChunk) : 1);
  const size_t smem = static_cast<size_t>(experts) * kSortWarps * 2;
  cudaFuncSetAttribute(expert_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxExperts * kSortWarps * 2);
  if (p.chunks > 1) {
    char *ws = static_cast<char *>(device_workspace(kScratchCounterBytes + static_cast<size_t>(p.chunks) * experts * 4, st));
    if (!ws) return BSIR_ERR_WORKSPACE;
    p.table = reinterpret_cast<int32_t *>(ws + kScratchCounterBytes);
    launch_pdl(expert_count_kernel, dim3(p.chunks), dim3(kSortThreads), 0, st, p);
    count_launch();
  }
  launch_pdl(expert_place_kernel, dim3(p.chunks), dim3(kSortThreads), smem, st, p);
  count_launch();
  return check_launch("expert_sort");
}

int32_t bsir_expert_dispatch(int32_t dtype, int64_t tokens, int64_t top_k, int64_t cols, const void *x, int64_t x_row_stride, const int32_t *slots,
                             int64_t out_rows, void *out, int64_t out_row_stride, void *stream) {
  clear_error();
  const int eb = dtype_bytes(dtype);
  if (eb == 0) return fail(BSIR_ERR_DTYPE, "expert_dispatch: dtype %d", dtype);
  if (int32_t rc = check_choice("expert_dispatch", tokens, top_k, cols, out_rows)) return rc;
  if (tokens == 0 || top_k == 0 || cols == 0) return BSIR_OK;
  if (!x || !slots || (!out && out_rows > 0)) return fail(BSIR_ERR_NULL, "expert_dispatch: null pointer");
  if (int32_t rc = check_stride("expert_dispatch", "x", tokens, cols, &x_row_stride)) return rc;
  if (int32_t rc = check_stride("expert_dispatch", "out", out_rows, cols, &out_row_stride)) return rc;
  if (!aligned_to(x, eb) || !aligned_to(out, eb) || !aligned_to(slots, 4)) return fail(BSIR_ERR_ALIGN, "expert_dispatch: misaligned");
  const int64_t out_bytes = span(out_rows, cols, out_row_stride, eb);
  if (overlap(x, span(tokens, cols, x_row_stride, eb), out, out_bytes) || overlap(slots, tokens * top_k * 4, out, out_bytes))
    return fail(BSIR_ERR_UNSUPPORTED, "expert_dispatch: out may not overlap x or slots");
  RowParams p{};
  p.tokens = tokens; p.top_k = static_cast<int>(top_k); p.rows = out_rows; p.slots = slots;
  p.x = x; p.out = out;
  p.err = device_error_word();
  if (!p.err) return fail(BSIR_ERR_WORKSPACE, "expert_dispatch: no device error word");
  cudaStream_t st = resolve_stream(stream);
  // the widest piece that bases, strides and the row's length are multiples of
  const int64_t row = cols * eb, xb = x_row_stride * eb, ob = out_row_stride * eb;
  int piece = 16;
  while (piece > eb && (!aligned_to(x, piece) || !aligned_to(out, piece) || xb % piece || ob % piece || row % piece)) piece >>= 1;
  p.cols = row / piece; p.xs = xb / piece; p.os = ob / piece;
  const dim3 grid = move_grid(tokens, ceil_div(p.cols, kMoveThreads * 4));
  switch (piece) {
    case 16: launch_pdl(expert_dispatch_kernel<uint4>, grid, dim3(kMoveThreads), 0, st, p); break;
    case 8: launch_pdl(expert_dispatch_kernel<uint64_t>, grid, dim3(kMoveThreads), 0, st, p); break;
    case 4: launch_pdl(expert_dispatch_kernel<uint32_t>, grid, dim3(kMoveThreads), 0, st, p); break;
    case 2: launch_pdl(expert_dispatch_kernel<uint16_t>, grid, dim3(kMoveThreads), 0, st, p); break;
    default: launch_pdl(expert_dispatch_kernel<uint8_t>, grid, dim3(kMoveThreads), 0, st, p); break;
  }
  count_launch();
  return check_launch("expert_dispatch");
}

int32_t bsir_expert_combine(int32_t dtype, int64_t tokens, int64_t top_k, int64_t cols, int64_t y_rows, const void *y, int64_t y_row_stride,
                            const int32_t *slots, int32_t weight_dtype, const void *weights, void *out, int64_t out_row_stride, void *stream) {
  clear_error();
  if (!dtype_is_float(dtype)) return fail(BSIR_ERR_DTYPE, "expert_combine: dtype %d (f32, f16, bf16)", dtype);
  if (weights && !dtype_is_float(weight_dtype)) return fail(BSIR_ERR_DTYPE, "expert_combine: weight dtype %d (f32, f16, bf16)", weight_dtype);
  if (int32_t rc = check_choice("expert_combine", tokens, top_k, cols, y_rows)) return rc;
  if (tokens == 0 || cols == 0) return BSIR_OK;
  if (!out || (top_k > 0 && !slots) || (top_k > 0 && y_rows > 0 && !y)) return fail(BSIR_ERR_NULL, "expert_combine: null pointer");
  if (int32_t rc = check_stride("expert_combine", "y", y_rows, cols, &y_row_stride)) return rc;
  if (int32_t rc = check_stride("expert_combine", "out", tokens, cols, &out_row_stride)) return rc;
  const int eb = dtype_bytes(dtype), wb = weights ? dtype_bytes(weight_dtype) : 0;
  if (!aligned_to(y, eb) || !aligned_to(out, eb) || !aligned_to(slots, 4) || (weights && !aligned_to(weights, wb)))
    return fail(BSIR_ERR_ALIGN, "expert_combine: misaligned");
  const int64_t out_bytes = span(tokens, cols, out_row_stride, eb);
  if (overlap(y, span(y_rows, cols, y_row_stride, eb), out, out_bytes) || overlap(slots, tokens * top_k * 4, out, out_bytes) ||
      overlap(weights, tokens * top_k * wb, out, out_bytes))
    return fail(BSIR_ERR_UNSUPPORTED, "expert_combine: out may not overlap an operand");
  RowParams p{};
  p.tokens = tokens; p.top_k = static_cast<int>(top_k); p.cols = cols; p.rows = y_rows; p.y = y; p.ys = y_row_stride;
  p.slots = slots; p.w = weights; p.w_dtype = weight_dtype; p.out = out; p.os = out_row_stride;
  p.err = device_error_word();
  if (!p.err) return fail(BSIR_ERR_WORKSPACE, "expert_combine: no device error word");
  const bool vec = (cols * eb) % 16 == 0 && rows_aligned(y, y_row_stride, eb) && rows_aligned(out, out_row_stride, eb);
  cudaStream_t st = resolve_stream(stream);
  switch (dtype) {
    case BSIR_F32: return launch_combine<BSIR_F32>(p, vec, st);
    case BSIR_F16: return launch_combine<BSIR_F16>(p, vec, st);
    default: return launch_combine<BSIR_BF16>(p, vec, st);
  }
}

int32_t bsir_expert_combine_grad(int32_t dtype, int64_t tokens, int64_t top_k, int64_t cols, int64_t y_rows, const void *dout,
                                 int64_t dout_row_stride, const void *y, int64_t y_row_stride, const int32_t *slots, int32_t weight_dtype,
                                 const void *weights, void *dy, int64_t dy_row_stride, float *dweights, void *stream) {
  clear_error();
  if (!dtype_is_float(dtype)) return fail(BSIR_ERR_DTYPE, "expert_combine_grad: dtype %d (f32, f16, bf16)", dtype);
  if (weights && !dtype_is_float(weight_dtype)) return fail(BSIR_ERR_DTYPE, "expert_combine_grad: weight dtype %d (f32, f16, bf16)", weight_dtype);
  if (int32_t rc = check_choice("expert_combine_grad", tokens, top_k, cols, y_rows)) return rc;
  if (tokens == 0 || top_k == 0) return BSIR_OK;
  if (!slots || !dweights || (cols > 0 && (!dout || (y_rows > 0 && (!y || !dy))))) return fail(BSIR_ERR_NULL, "expert_combine_grad: null pointer");
  if (int32_t rc = check_stride("expert_combine_grad", "dout", tokens, cols, &dout_row_stride)) return rc;
  if (int32_t rc = check_stride("expert_combine_grad", "y", y_rows, cols, &y_row_stride)) return rc;
  if (int32_t rc = check_stride("expert_combine_grad", "dy", y_rows, cols, &dy_row_stride)) return rc;
  const int eb = dtype_bytes(dtype), wb = weights ? dtype_bytes(weight_dtype) : 0;
  if (!aligned_to(dout, eb) || !aligned_to(y, eb) || !aligned_to(dy, eb) || !aligned_to(slots, 4) || !aligned_to(dweights, 4) ||
      (weights && !aligned_to(weights, wb)))
    return fail(BSIR_ERR_ALIGN, "expert_combine_grad: misaligned");
  const int64_t n = tokens * top_k;
  struct { const void *p; int64_t bytes; } in[4] = {{dout, span(tokens, cols, dout_row_stride, eb)}, {y, span(y_rows, cols, y_row_stride, eb)},
                                                    {slots, n * 4}, {weights, n * wb}};
  const int64_t dy_bytes = span(y_rows, cols, dy_row_stride, eb);
  for (const auto &i : in)
    if (overlap(i.p, i.bytes, dy, dy_bytes) || overlap(i.p, i.bytes, dweights, n * 4))
      return fail(BSIR_ERR_UNSUPPORTED, "expert_combine_grad: a gradient may not overlap an operand");
  if (overlap(dy, dy_bytes, dweights, n * 4)) return fail(BSIR_ERR_UNSUPPORTED, "expert_combine_grad: the gradients may not overlap");
  RowParams p{};
  p.tokens = tokens; p.top_k = static_cast<int>(top_k); p.cols = cols; p.rows = y_rows; p.x = dout; p.xs = dout_row_stride;
  p.y = y; p.ys = y_row_stride; p.slots = slots; p.w = weights; p.w_dtype = weight_dtype; p.dy = dy; p.dys = dy_row_stride; p.dw = dweights;
  p.err = device_error_word();
  if (!p.err) return fail(BSIR_ERR_WORKSPACE, "expert_combine_grad: no device error word");
  const bool vec = (cols * eb) % 16 == 0 && rows_aligned(dout, dout_row_stride, eb) && rows_aligned(y, y_row_stride, eb) &&
                   rows_aligned(dy, dy_row_stride, eb);
  cudaStream_t st = resolve_stream(stream);
  switch (dtype) {
    case BSIR_F32: return launch_combine_grad<BSIR_F32>(p, vec, st);
    case BSIR_F16: return launch_combine_grad<BSIR_F16>(p, vec, st);
    default: return launch_combine_grad<BSIR_BF16>(p, vec, st);
  }
}

}  // extern "C"
