// Eviction by accumulated attention weight. Of the first n places of a cache each KV head (or all
// heads together, by the sum of their weights) keeps `keep`: the protected positions and then those
// of the largest weight, equal weights in the order of their places, a NaN below every number. The
// kept tokens behind place `keep` move, in order, into the places before it that were given up, so
// no row is read after it has been overwritten, as few rows move as can, and keys that carry their
// rotary position stay as they are (attention does not mind the order).
//
// evict_select_kernel: one cluster of CTAs per choice (a KV head, or all of them). A radix select over
// order-preserving 32-bit keys finds the smallest kept key, 8 bits a pass: each CTA counts its own
// run of places in shared memory, and after a cluster barrier every CTA adds up the cluster's counts
// through distributed shared memory. The keys stay in shared memory between passes where they fit.
// A last scan in the order of the places writes the compacted weights and positions, and lists the
// places to fill and the places to move. evict_move_kernel moves the pool rows.
//
// Bound by HBM: the weights are read once; per moved token and head two packed rows and their scales
// are read and written.
#include <cooperative_groups.h>

#include "cache_ops.cuh"

namespace cg = cooperative_groups;

namespace kvb {
namespace {

constexpr int kCluster = 8;
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 256;
constexpr int kMaxCached = 48 * 1024;  // keys a CTA keeps in shared memory

// Larger key = kept first. -0 counts as 0; a NaN ranks below every number.
__device__ __forceinline__ unsigned weight_key(float w) {
  if (w != w) return 0u;
  const unsigned b = __float_as_uint(w + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ unsigned place_key(const EvictArgs& a, int list, int place) {
  const int pos = a.positions[list * a.positions_stride + place];
  if (pos < a.sink || pos >= a.recent_from) return 0xFFFFFFFFu;
  float w;
  if (a.shared) {
    double sum = 0.0;
    for (int h = 0; h < a.kvh; ++h) sum += static_cast<double>(a.weights[h * a.weights_stride + place]);
    w = static_cast<float>(sum);
  } else {
    w = a.weights[list * a.weights_stride + place];
  }
  return weight_key(w);
}

struct Counts {  // places of a run by (key above or equal the border, before or behind `keep`)
  int above_early, equal_early, above_late, equal_late;
};

__device__ __forceinline__ Counts operator+(const Counts& x, const Counts& y) {
  return {x.above_early + y.above_early, x.equal_early + y.equal_early, x.above_late + y.above_late,
          x.equal_late + y.equal_late};
}

__global__ void __launch_bounds__(kThreads) evict_select_kernel(const EvictArgs a, int run, int cached) {
  extern __shared__ unsigned keys[];  // [run] when cached
  __shared__ unsigned hist[2][kBins];
  __shared__ unsigned total[kBins];
  __shared__ Counts warp_counts[kWarps];
  __shared__ Counts cta_counts;
  __shared__ unsigned found[2];  // digit, keys above it
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int list = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = min(a.n, rank * run), last = min(a.n, first + run);

  pdl_wait();
  pdl_launch();
  const auto key_at = [&](int i) { return cached ? keys[i - first] : place_key(a, list, i); };
  if (cached)
    for (int i = first + static_cast<int>(threadIdx.x); i < last; i += kThreads)
      keys[i - first] = place_key(a, list, i);

  // The keep-th largest key, digit by digit; `need` = how many of the keys with this prefix to keep.
  unsigned prefix = 0, need = static_cast<unsigned>(a.keep);
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    unsigned* mine = hist[pass & 1];
    for (int b = threadIdx.x; b < kBins; b += kThreads) mine[b] = 0;
    __syncthreads();
    for (int i = first + static_cast<int>(threadIdx.x); i < last; i += kThreads) {
      const unsigned k = key_at(i);
      if (pass == 0 || (k >> (shift + 8)) == prefix) atomicAdd(&mine[k >> shift & 255u], 1u);
    }
    cluster.sync();
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
      unsigned sum = 0;
      for (int r = 0; r < kCluster; ++r) sum += *cluster.map_shared_rank(&mine[b], r);
      total[b] = sum;
    }
    __syncthreads();
    if (warp == 0) {  // lane l: bins 255 - 8 l downwards
      unsigned own[8], sum = 0;
      for (int j = 0; j < 8; ++j) sum += own[j] = total[255 - 8 * lane - j];
      unsigned before = sum;
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
      }
      before -= sum;
      if (before < need && need <= before + sum) {
        int j = 0;
        while (before + own[j] < need) before += own[j++];
        found[0] = 255 - 8 * lane - j;
        found[1] = before;
      }
    }
    __syncthreads();
    prefix = prefix << 8 | found[0];
    need -= found[1];
    // hist[pass & 1] is written again two passes on, behind the next pass's cluster barrier
  }
  const unsigned border = prefix;  // kept: keys above it, and the first `need` equal to it

  // Warp w counts its own run of places, 32 at a time in their order.
  const int per_warp = (run + kWarps * 32 - 1) / (kWarps * 32) * 32;
  const int wfirst = min(last, first + warp * per_warp), wlast = min(last, wfirst + per_warp);
  Counts c{0, 0, 0, 0};
  for (int i = wfirst + lane; i - lane < wlast; i += 32) {
    const unsigned k = i < wlast ? key_at(i) : 0u;
    const bool in = i < wlast, early = i < a.keep;
    c.above_early += __popc(__ballot_sync(0xffffffffu, in && early && k > border));
    c.equal_early += __popc(__ballot_sync(0xffffffffu, in && early && k == border));
    c.above_late += __popc(__ballot_sync(0xffffffffu, in && !early && k > border));
    c.equal_late += __popc(__ballot_sync(0xffffffffu, in && !early && k == border));
  }
  if (lane == 0) warp_counts[warp] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    Counts sum{0, 0, 0, 0};
    for (int w = 0; w < kWarps; ++w) {
      const Counts own = warp_counts[w];
      warp_counts[w] = sum;
      sum = sum + own;
    }
    cta_counts = sum;
  }
  cluster.sync();
  Counts before = warp_counts[warp];
  for (int r = 0; r < rank; ++r) before = before + *cluster.map_shared_rank(&cta_counts, r);

  // Ranks in the order of the places: equal keys, places to fill, places to move.
  int equals = before.equal_early + before.equal_late;
  const int want = static_cast<int>(need);
  // of the equal keys before this run the first `want` are kept; the early ones come first
  const int kept_early = before.above_early + min(before.equal_early, want);
  int late = before.above_late + min(equals, want) - min(before.equal_early, want);
  int hole = min(wfirst, a.keep) - kept_early;
  const int lists = a.shared ? a.kvh : 1;  // heads this choice is for
  int32_t* holes = a.holes + static_cast<long long>(list) * a.keep;
  int32_t* movers = a.movers + static_cast<long long>(list) * (a.n - a.keep);
  for (int i = wfirst + lane; i - lane < wlast; i += 32) {
    const bool in = i < wlast, early = i < a.keep;
    const unsigned k = in ? key_at(i) : 0u;
    const unsigned below = (1u << lane) - 1u;
    const unsigned eq = __ballot_sync(0xffffffffu, in && k == border);
    const bool kept = in && (k > border || (k == border && equals + __popc(eq & below) < want));
    equals += __popc(eq);
    const unsigned fill = __ballot_sync(0xffffffffu, in && early && !kept);
    const unsigned move = __ballot_sync(0xffffffffu, kept && !early);
    if (in && early && !kept) holes[hole + __popc(fill & below)] = i;
    if (kept && !early) movers[late + __popc(move & below)] = i;
    hole += __popc(fill);
    late += __popc(move);
    if (in)
      for (int j = 0; j < lists; ++j) {
        const int h = list + j;
        const long long to = static_cast<long long>(h) * a.columns + i;
        if (early && kept) {
          a.new_weights[to] = a.weights[h * a.weights_stride + i];
          a.new_positions[to] = a.positions[h * a.positions_stride + i];
        } else if (!early) {
          a.new_weights[to] = 0.f;
          a.new_positions[to] = -1;
        }
      }
  }
  if (rank == kCluster - 1) {  // the columns behind the cache's length
    for (int i = a.n + static_cast<int>(threadIdx.x); i < a.columns; i += kThreads)
      for (int j = 0; j < lists; ++j) {
        a.new_weights[static_cast<long long>(list + j) * a.columns + i] = 0.f;
        a.new_positions[static_cast<long long>(list + j) * a.columns + i] = -1;
      }
    if (warp == kWarps - 1 && lane == 0) a.counts[list] = late;  // the last run's end: all movers
    if (list == 0)
      for (int b = threadIdx.x; b < a.n_sel; b += kThreads) {
        const int blk = a.table ? a.table[b] : b;
        if (blk >= 0 && blk < a.n_pool)
          a.valid[blk] = static_cast<int>(max(0ll, min(static_cast<long long>(a.bt),
                                                       a.keep - static_cast<long long>(b) * a.bt)));
        else if (a.status)
          atomicOr(a.status, kDevBadBlockIndex);
      }
  }
  cluster.sync();  // the lists are complete (and no CTA leaves while its counts are read)
  const int moved = a.counts[list];
  for (int j = rank * kThreads + threadIdx.x; j < moved; j += kCluster * kThreads) {
    const int to = holes[j], from = movers[j];
    for (int i = 0; i < lists; ++i) {
      const int h = list + i;
      a.new_weights[static_cast<long long>(h) * a.columns + to] = a.weights[h * a.weights_stride + from];
      a.new_positions[static_cast<long long>(h) * a.columns + to] =
          a.positions[h * a.positions_stride + from];
    }
  }
}

// Pool row (in tokens) of a place, or -1 for a refused block.
__device__ __forceinline__ long long token_row(const EvictArgs& a, int place) {
  const int slot = place / a.bt;
  const int blk = a.table ? a.table[slot] : slot;
  if (blk < 0 || blk >= a.n_pool) return -1;
  return static_cast<long long>(blk) * a.bt + (place - slot * a.bt);
}

// One item: `unit` bytes of one moved row, of codes or scales, of K or V. With one choice for all
// heads a row is a whole token (kvh heads are contiguous).
template <typename U, typename S>
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictArgs a, int code_units,
                                                         int scale_units) {
  const int list = blockIdx.y, heads = a.shared ? 1 : a.kvh;
  const int units = 2 * (code_units + scale_units);
  pdl_wait();
  pdl_launch();
  const int32_t* holes = a.holes + static_cast<long long>(list) * a.keep;
  const int32_t* movers = a.movers + static_cast<long long>(list) * (a.n - a.keep);
  const long long items = static_cast<long long>(a.counts[list]) * units;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < items; i += gridDim.x * 256ll) {
    const int j = static_cast<int>(i / units);
    int u = static_cast<int>(i - static_cast<long long>(j) * units);
    const int kv = u >= code_units + scale_units;
    if (kv) u -= code_units + scale_units;
    const long long from = token_row(a, movers[j]), to = token_row(a, holes[j]);
    if (from < 0 || to < 0) continue;
    if (u < code_units) {
      U* p = reinterpret_cast<U*>(a.packed[kv]);
      p[(to * heads + list) * code_units + u] = p[(from * heads + list) * code_units + u];
    } else {
      u -= code_units;
      S* p = reinterpret_cast<S*>(a.scales[kv]);
      p[(to * heads + list) * scale_units + u] = p[(from * heads + list) * scale_units + u];
    }
  }
}

template <typename U, typename S>
cudaError_t move_as(const EvictArgs& a, int code_bytes, int scale_bytes, cudaStream_t s) {
  const int lists = a.shared ? 1 : a.kvh;
  return launch_pdl(evict_move_kernel<U, S>, dim3((148 * 8 + lists - 1) / lists, lists), 256, 0, s, a,
                    code_bytes / static_cast<int>(sizeof(U)),
                    scale_bytes / static_cast<int>(sizeof(S)));
}

template <typename U>
cudaError_t move_codes(const EvictArgs& a, int code_bytes, int scale_bytes, cudaStream_t s) {
  const uintptr_t sp = reinterpret_cast<uintptr_t>(a.scales[0]) | reinterpret_cast<uintptr_t>(a.scales[1]) | scale_bytes;
  if (sp % 16 == 0) return move_as<U, uint4>(a, code_bytes, scale_bytes, s);
  if (sp % 8 == 0) return move_as<U, uint2>(a, code_bytes, scale_bytes, s);
  if (sp % 4 == 0) return move_as<U, uint32_t>(a, code_bytes, scale_bytes, s);
  return move_as<U, uint16_t>(a, code_bytes, scale_bytes, s);
}

}  // namespace

cudaError_t launch_evict(const EvictArgs& a, cudaStream_t s) {
  const int lists = a.shared ? 1 : a.kvh;
  const int run = ((a.n + kCluster - 1) / kCluster + 31) / 32 * 32;
  const int cached = run <= kMaxCached;
  const size_t smem = cached ? run * sizeof(unsigned) : 0;
  cudaError_t e = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kMaxCached * sizeof(unsigned));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kCluster, lists, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kCluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, evict_select_kernel, a, run, cached);
  if (e != cudaSuccess) return e;
  const int heads = a.shared ? a.kvh : 1;
  const int code_bytes = heads * a.packed_dim, scale_bytes = heads * a.groups * 2;
  const uintptr_t cp = reinterpret_cast<uintptr_t>(a.packed[0]) | reinterpret_cast<uintptr_t>(a.packed[1]) | code_bytes;
  if (cp % 16 == 0) return move_codes<uint4>(a, code_bytes, scale_bytes, s);
  if (cp % 4 == 0) return move_codes<uint32_t>(a, code_bytes, scale_bytes, s);
  return move_codes<uint8_t>(a, code_bytes, scale_bytes, s);
}

}  // namespace kvb
