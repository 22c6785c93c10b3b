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

#include <atomic>

namespace bsir {
namespace {

// ------------------------------------------------------------------------------------------------ sort
// A stable counting sort in one launch: one CTA for up to 4096 choices, a cluster of eight for up to 16384, of sixteen for
// more (65536 choices of 128 experts: 8.2 us, 10.7 by eight; 524288: 48 and 89).  Each of the cluster's warps owns a run of consecutive choices and goes over it 32 at a time: the lanes with one expert find each
// other by ballots over the bits of its number (match.any takes about 70 cycles of the SM, for whatever warp), and a
// choice's rank among them is a popcount.  That leaves every warp's count of every expert; the counts of the warps
// before it, of the CTAs before it (read through distributed shared memory) and of the experts before its own add up to
// a choice's row.  Runs of up to 32 * kSortGroups choices stay in registers with their ranks, longer ones are gone over
// twice.  No scratch in global memory, and no atomics.
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortOneCta = 4096;
constexpr int kSortEight = 16384;
constexpr int kMaxExperts = 1024;

struct SortParams {
  const void *ids;
  int64_t n;                  // choices
  int64_t run;                // choices of a warp, a multiple of 32
  int experts;
  int wide;                   // ids are int64
  int ctas;                   // of the cluster
  int32_t *offsets, *slots;
};
__device__ __forceinline__ int load_id(const SortParams &p, int64_t i, int64_t end) {
  if (i >= end) return -1;
  if (p.wide) {
    const long long v = static_cast<const long long *>(p.ids)[i];
    return v >= 0 && v < p.experts ? static_cast<int>(v) : -1;
  }
  const int v = static_cast<const int *>(p.ids)[i];
  return v >= 0 && v < p.experts ? v : -1;
}

// the lanes of the warp whose expert is this lane's (masked choices are one more expert)
__device__ __forceinline__ unsigned same_expert(int id, int experts, int bits) {
  const unsigned key = static_cast<unsigned>(id < 0 ? experts : id);
  unsigned peers = 0xffffffffu;
  for (int b = 0; b < bits; ++b) {
    const unsigned set = __ballot_sync(0xffffffffu, key >> b & 1u);
    peers &= key >> b & 1u ? set : ~set;
  }
  return peers;
}

// exclusive prefix sum of one value a thread over the whole CTA; *total the sum
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

__device__ __forceinline__ void cluster_barrier() {            // warps may come to it in parts
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ int load_peer(const int *own, int cta) {       // the same shared-memory word in another CTA
  uint32_t addr = static_cast<uint32_t>(__cvta_generic_to_shared(own)), peer;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(addr), "r"(cta));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(peer) : "memory");
  return v;
}

constexpr int kSortGroups = 8;                   // of 32 choices that a warp keeps in registers
template <bool KEEP>
__global__ void __launch_bounds__(kSortThreads) expert_sort_kernel(SortParams p) {
  extern __shared__ int warp_count[];            // [kSortWarps][experts]: a warp's choices of an expert, then its next row
  __shared__ int mine_s[kMaxExperts];            // this CTA's choices of an expert
  __shared__ int warp_sum_s[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x;                   // the grid is one cluster
  for (int i = tid; i < p.experts * kSortWarps; i += kSortThreads) warp_count[i] = 0;
  pdl_launch_dependents();
  pdl_wait();
  __syncthreads();
  const int64_t first = (static_cast<int64_t>(rank) * kSortWarps + warp) * p.run;
  const int64_t end = first + p.run < p.n ? first + p.run : p.n;
  const unsigned below = (1u << lane) - 1u;
  const int bits = 32 - __clz(p.experts);
  int *own = warp_count + warp * p.experts;
  int id[kSortGroups], ahead[kSortGroups];       // KEEP: the warp's choices, and how many of their expert come before them
  if constexpr (KEEP) {
#pragma unroll
    for (int u = 0; u < kSortGroups; ++u) id[u] = load_id(p, first + u * 32 + lane, end);
#pragma unroll
    for (int u = 0; u < kSortGroups; ++u) {
      if (first + u * 32 >= end) break;
      const unsigned peers = same_expert(id[u], p.experts, bits);
      ahead[u] = id[u] < 0 ? 0 : own[id[u]] + __popc(peers & below);
      __syncwarp();
      if (id[u] >= 0 && (peers & below) == 0) own[id[u]] += __popc(peers);
      __syncwarp();
    }
  } else {
    for (int64_t i0 = first; i0 < end; i0 += 128) {          // four groups of 32 in flight
#pragma unroll
      for (int u = 0; u < 4; ++u) id[u] = load_id(p, i0 + u * 32 + lane, end);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const unsigned peers = same_expert(id[u], p.experts, bits);
        if (id[u] >= 0 && (peers & below) == 0) own[id[u]] += __popc(peers);
        __syncwarp();
      }
    }
  }
  __syncthreads();
  int mine = 0;
  if (tid < p.experts) {
#pragma unroll 8
    for (int w = 0; w < kSortWarps; ++w) mine += warp_count[w * p.experts + tid];
    mine_s[tid] = mine;
  }
  if (p.ctas > 1) cluster_barrier();
  int earlier = 0, all = mine;
  if (p.ctas > 1 && tid < p.experts) {
    all = 0;
    for (int c = 0; c < p.ctas; ++c) {
      const int v = load_peer(&mine_s[tid], c);
      if (c < rank) earlier += v;
      all += v;
    }
  }
  int total;
  const int start = cta_prefix(all, warp_sum_s, &total);
  if (tid < p.experts) {
    int next = start + earlier;
#pragma unroll 8
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = warp_count[w * p.experts + tid];
      warp_count[w * p.experts + tid] = next;
      next += c;
    }
    if (rank == 0) p.offsets[tid] = start;
  }
  if (rank == 0 && tid == 0) p.offsets[p.experts] = total;
  __syncthreads();
  if constexpr (KEEP) {
#pragma unroll
    for (int u = 0; u < kSortGroups; ++u) {
      const int64_t i = first + u * 32 + lane;
      if (i < end) p.slots[i] = id[u] < 0 ? -1 : own[id[u]] + ahead[u];
    }
  } else {
    for (int64_t i0 = first; i0 < end; i0 += 128) {
#pragma unroll
      for (int u = 0; u < 4; ++u) id[u] = load_id(p, i0 + u * 32 + lane, end);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const unsigned peers = same_expert(id[u], p.experts, bits);
        const int at = id[u] < 0 ? 0 : id[u];
        const int row = own[at] + __popc(peers & below);
        __syncwarp();
        if (id[u] >= 0 && (peers & below) == 0) own[at] += __popc(peers);
        __syncwarp();
        const int64_t i = i0 + u * 32 + lane;
        if (i < end) p.slots[i] = id[u] < 0 ? -1 : row;
      }
    }
  }
  if (p.ctas > 1) cluster_barrier();             // a peer may still be reading this CTA's counts
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

// One CTA per token, four choices at a time: y's rows are read once, dy's written once, dout's once for the four; the dot
// products meet across the warps in a fixed order.  (64k rows of 4096 bf16: 180 us; eight choices at a time 267, dout kept
// in registers for eight 194.)
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

// Whether the current device runs a cluster of sixteen of the sort's CTAs (more than the eight that every one does; a GPC
// has to have as many SMs).  Asked once per device.
bool sixteen_at_once() {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices];                        // 1: no, 2: yes
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device >= kDevices) return false;
  int answer = known[device].load(std::memory_order_relaxed);
  if (answer == 0) {
    int n = 1;
    for (auto kernel : {expert_sort_kernel<true>, expert_sort_kernel<false>}) {
      constexpr int kSmem = kMaxExperts * kSortWarps * 4;
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(16);
      cfg.blockDim = dim3(kSortThreads);
      cfg.dynamicSmemBytes = kSmem;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = 16;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      int fits = 0;
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess ||
          cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
          cudaOccupancyMaxActiveClusters(&fits, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return false;               // not remembered: the next call asks again
      }
      n = fits < n ? fits : n;
    }
    answer = n > 0 ? 2 : 1;
    known[device].store(answer, std::memory_order_relaxed);
  }
  return answer == 2;
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
  p.ctas = n <= kSortOneCta ? 1 : n <= kSortEight || !sixteen_at_once() ? 8 : 16;
  p.run = ceil_div(ceil_div(n, static_cast<int64_t>(p.ctas) * kSortWarps), 32) * 32;
  const size_t smem = static_cast<size_t>(experts) * kSortWarps * 4;
  auto kernel = p.run <= 32 * kSortGroups ? expert_sort_kernel<true> : expert_sort_kernel<false>;
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxExperts * kSortWarps * 4);
  if (p.ctas > 1) launch_pdl_cluster(kernel, dim3(p.ctas), dim3(kSortThreads), smem, st, p.ctas, p);
  else launch_pdl(kernel, dim3(1), dim3(kSortThreads), smem, st, p);
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
