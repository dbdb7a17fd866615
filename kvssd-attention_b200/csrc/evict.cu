// Eviction by accumulated attention weight. Of the first n places of a cache each KV head (or all
// heads together, by the sum of their weights) keeps `keep`: the protected positions and then those
// of the largest weight, equal weights in the order of their places, a NaN below every number. The
// kept tokens behind place `keep` move, in order, into the places before it that were given up, so
// no row is read after it has been overwritten, as few rows move as can, and keys that carry their
// rotary position stay as they are (attention does not mind the order).
//
// Selection: one cluster of CTAs per choice (a KV head, or all of them). A radix select over
// order-preserving 32-bit keys finds the smallest kept key, a digit a pass: each CTA counts its own run
// of places in shared memory, and after a cluster barrier every CTA adds up the cluster's counts
// through distributed shared memory. A last scan in the order of the places copies the weights and
// positions that stay and lists the places to fill and the places to move (their numbers are equal).
// evict_select_kernel keeps each thread's run of consecutive keys in registers;
// evict_select_long_kernel is the form for caches that do not fit (keys in shared memory, or in scratch). evict_move_kernel then moves the
// pool rows with their weights and positions, on all SMs.
//
// Bound by HBM: the weights are read once; per moved token and head two packed rows and their scales
// are read and written. 131072 to 65536 tokens x 8 heads x 128 INT4: 53 us, 27 of them the selection
// (its three rounds) and 26 the moves (rows of 64 bytes; floor of all 13.4); 1048576 to 524288: 511 us,
// one choice for all heads 661.
#include <cooperative_groups.h>

#include "cache_ops.cuh"

namespace cg = cooperative_groups;

namespace kvb {
namespace {

constexpr int kMaxCluster = 8;  // larger ones are not portable, and few fit beside each other
constexpr int kLongCluster = kMaxCluster;
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

// Which digit of the keys holds the `need`-th largest, and how many keys lie above it: from the
// cluster's counts of every digit. All threads; `found` is shared.
__device__ __forceinline__ void find_digit(const unsigned* total, unsigned need, unsigned* found) {
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {  // lane l: bins 255 - 8 l downwards
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
}

// The compacted cache's valid counts, by the threads of one CTA.
__device__ __forceinline__ void write_valid_counts(const EvictArgs& a) {
  for (int b = threadIdx.x; b < a.n_sel; b += kThreads) {
    const int blk = a.table ? a.table[b] : b;
    if (blk >= 0 && blk < a.n_pool)
      a.valid[blk] = static_cast<int>(max(0ll, min(static_cast<long long>(a.bt),
                                                   a.keep - static_cast<long long>(b) * a.bt)));
    else if (a.status)
      atomicOr(a.status, kDevBadBlockIndex);
  }
}

// The two halves of a cluster barrier.
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct Counts {  // places of a run by (key above or equal the border, before or behind `keep`)
  int above_early, equal_early, above_late, equal_late;
};

__device__ __forceinline__ Counts operator+(const Counts& x, const Counts& y) {
  return {x.above_early + y.above_early, x.equal_early + y.equal_early, x.above_late + y.above_late,
          x.equal_late + y.equal_late};
}

// x in FP64, by its bits: the conversion instruction is an eighth as fast as the addition.
__device__ __forceinline__ double widen(float x) {
  const unsigned b = __float_as_uint(x), m = b & 0x7FFFFFFFu;
  if (m - 0x00800000u < 0x7F000000u)  // neither zero, subnormal, infinite nor NaN
    return __hiloint2double(static_cast<int>((b & 0x80000000u) | ((m >> 3) + 0x38000000u)),
                            static_cast<int>(b << 29));
  return m == 0 ? 0.0 : static_cast<double>(x);
}

// V consecutive numbers, in one access.
template <int V, typename T>
struct alignas(sizeof(T) * V) Run {
  T e[V];
};

// Keys of the places [first, last) to `keys`, and their weights and positions to their new places. A
// thread has kBatch runs in flight, of consecutive steps or, when SHARED, of consecutive heads (all
// loads come before the stores, which the compiler cannot tell apart).
template <int E, int V, bool SHARED>
__device__ __forceinline__ void load_places(const EvictArgs& a, int list, int first, int last, unsigned* keys) {
  using Weights = Run<V, float>;
  using Positions = Run<V, int32_t>;
  constexpr int kBatch = SHARED || E / V >= 4 ? 4 : E / V, kSteps = SHARED ? 1 : kBatch;
  for (int base = first; base < last; base += kThreads * V * kSteps) {
    double sum[SHARED ? V : 1] = {};
    Positions own;  // of a shared choice: those of head 0
    for (int h0 = list; h0 < (SHARED ? a.kvh : list + 1); h0 += kBatch) {
      Weights w[kBatch];
      Positions p[kBatch];
#pragma unroll
      for (int s = 0; s < kBatch; ++s) {
        const int h = SHARED ? h0 + s : list;
        const int i = base + ((SHARED ? 0 : s) * kThreads + static_cast<int>(threadIdx.x)) * V;
        const float* from_w = a.weights + h * a.weights_stride + i;
        const int32_t* from_p = a.positions + h * a.positions_stride + i;
        if (SHARED && h >= a.kvh) continue;
        if (i + V <= last) {
          w[s] = *reinterpret_cast<const Weights*>(from_w);
          p[s] = *reinterpret_cast<const Positions*>(from_p);
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (i + k < last) w[s].e[k] = from_w[k], p[s].e[k] = from_p[k];
        }
      }
#pragma unroll
      for (int s = 0; s < kBatch; ++s) {
        const int h = SHARED ? h0 + s : list;
        const int i = base + ((SHARED ? 0 : s) * kThreads + static_cast<int>(threadIdx.x)) * V;
        if (SHARED && h >= a.kvh) continue;
        if constexpr (SHARED) {
          if (h == list) own = p[s];
#pragma unroll
          for (int k = 0; k < V; ++k) sum[k] += widen(w[s].e[k]);
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (i + k < last)
              keys[i + k - first] = p[s].e[k] < a.sink || p[s].e[k] >= a.recent_from ? 0xFFFFFFFFu : weight_key(w[s].e[k]);
        }
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (i + k >= a.keep) w[s].e[k] = 0.f, p[s].e[k] = -1;
        const long long to = static_cast<long long>(h) * a.columns + i;
        if (i + V <= last) {
          *reinterpret_cast<Weights*>(a.new_weights + to) = w[s];
          *reinterpret_cast<Positions*>(a.new_positions + to) = p[s];
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (i + k < last) a.new_weights[to + k] = w[s].e[k], a.new_positions[to + k] = p[s].e[k];
        }
      }
    }
    if constexpr (SHARED) {
      const int i = base + static_cast<int>(threadIdx.x) * V;
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (i + k < last)
          keys[i + k - first] = own.e[k] < a.sink || own.e[k] >= a.recent_from ? 0xFFFFFFFFu : weight_key(static_cast<float>(sum[k]));
    }
  }
}

__global__ void __launch_bounds__(kThreads) evict_select_long_kernel(const EvictArgs a, int run, int cached, int vectors) {
  extern __shared__ __align__(16) unsigned in_shared[];  // the run's keys when cached; else in scratch
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
  unsigned* keys = cached ? in_shared : a.keys + static_cast<long long>(list) * a.n + first;
  if (a.shared) {
    if (vectors) load_places<16, 4, true>(a, list, first, last, keys);
    else load_places<16, 1, true>(a, list, first, last, keys);
  } else {
    if (vectors) load_places<16, 4, false>(a, list, first, last, keys);
    else load_places<16, 1, false>(a, list, first, last, keys);
  }
  const auto key_at = [&](int i) { return keys[i - first]; };

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
      for (int r = 0; r < kLongCluster; ++r) sum += *cluster.map_shared_rank(&mine[b], r);
      total[b] = sum;
    }
    __syncthreads();
    find_digit(total, need, found);
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
  }
  if (rank == kLongCluster - 1) {  // the columns behind the cache's length
    for (int i = a.n + static_cast<int>(threadIdx.x); i < a.columns; i += kThreads)
      for (int j = 0; j < lists; ++j) {
        a.new_weights[static_cast<long long>(list + j) * a.columns + i] = 0.f;
        a.new_positions[static_cast<long long>(list + j) * a.columns + i] = -1;
      }
    if (warp == kWarps - 1 && lane == 0) a.counts[list] = late;  // the last run's end: all movers
    if (list == 0) write_valid_counts(a);
  }
  cluster.sync();  // no CTA leaves while its counts are read
}

// The same for up to cluster * kThreads * E places: each CTA has a run of up to kThreads * E of them, and
// thread t of it holds the keys of the E places from t * E on in that run. Digits of 11, 11 and 10 bits: three rounds of counting, barrier, adding up
// and searching at about 3 us each, of which the counting is the smallest part. The weights and
// positions are written to their new places as soon as they are read (evict_move_kernel overwrites the
// places to fill), and the lists go through shared memory, so that their stores are whole lines.
constexpr int kDigits = 2048;

template <int E>
__global__ void __launch_bounds__(kThreads) evict_select_kernel(const EvictArgs a, int run, int vectors) {
  extern __shared__ __align__(16) unsigned dynamic[];  // kThreads * E keys, later places; two histograms
  __shared__ int2 warp_counts[kWarps];
  __shared__ unsigned warp_totals[kWarps];
  __shared__ Counts cta_counts;
  __shared__ unsigned found[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), ranks = static_cast<int>(cluster.num_blocks());
  const int list = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int cta_first = min(rank * run, a.n), cta_last = min(cta_first + run, a.n);
  const int first = cta_first + static_cast<int>(threadIdx.x) * E;
  const int lists = a.shared ? a.kvh : 1;  // heads this choice is for
  const int own = max(0, min(E, cta_last - first));       // places this thread holds
  const int split = min(max(a.keep - first, 0), own);     // those before `keep`

  unsigned* digits = dynamic + kThreads * E;
  for (int i = threadIdx.x; i < kDigits; i += kThreads) digits[i] = 0;
  pdl_wait();
  pdl_launch();
  // the CTA's places in order of the threads, V a thread and step: keys to shared memory, statistics
  // to their new places
  if (a.shared) {
    if (vectors) load_places<E, 4, true>(a, list, cta_first, cta_last, dynamic);
    else load_places<E, 1, true>(a, list, cta_first, cta_last, dynamic);
  } else {
    if (vectors) load_places<E, 4, false>(a, list, cta_first, cta_last, dynamic);
    else load_places<E, 1, false>(a, list, cta_first, cta_last, dynamic);
  }
  for (int i = 0; i < lists; ++i)  // the columns behind the cache's places
    for (int k = a.n + rank * kThreads + static_cast<int>(threadIdx.x); k < a.columns; k += ranks * kThreads) {
      a.new_weights[static_cast<long long>(list + i) * a.columns + k] = 0.f;
      a.new_positions[static_cast<long long>(list + i) * a.columns + k] = -1;
    }
  __syncthreads();
  unsigned keys[E];
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    const uint4 four = *reinterpret_cast<const uint4*>(dynamic + threadIdx.x * E + e);
    keys[e] = four.x, keys[e + 1] = four.y, keys[e + 2] = four.z, keys[e + 3] = four.w;
  }

  unsigned prefix = 0, need = static_cast<unsigned>(a.keep);
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    unsigned* mine = digits + (pass & 1) * kDigits;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < own && (pass == 0 || keys[e] >> (shift + bits & 31) == prefix))
        atomicAdd(&mine[keys[e] >> shift & ((1u << bits) - 1u)], 1u);
    cluster.sync();
    // thread t: digits 2047 - 2 t and the one below, over the cluster
    unsigned* other = digits + (pass + 1 & 1) * kDigits;
    const int top = kDigits - 2 - 2 * static_cast<int>(threadIdx.x);
    unsigned high = 0, low = 0;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r)  // unrolled: the remote loads overlap
      if (r < ranks) {
        const uint2 two = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(&mine[top], r));
        low += two.x;
        high += two.y;
      }
    // the other buffer is free: the barrier above ended the reads of the pass before
    *reinterpret_cast<uint2*>(&other[top]) = make_uint2(0, 0);
    unsigned before = high + low;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += up;
    }
    if (lane == 31) warp_totals[warp] = before;
    __syncthreads();
    unsigned upto = warp_totals[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    before += __shfl_sync(0xffffffffu, upto, warp) - warp_totals[warp] - high - low;
    if (before < need && need <= before + high + low) {  // one thread of the CTA
      const bool in_high = need <= before + high;
      found[0] = top + in_high;
      found[1] = in_high ? before : before + high;
    }
    __syncthreads();
    prefix = prefix << bits | found[0];
    need -= found[1];
  }
  const unsigned border = prefix;  // kept: keys above it, and the first `need` equal to it
  const int want = static_cast<int>(need);

  // counts of this thread's places, above | equal << 16 (a CTA has at most 2^14 places), summed over
  // the places before
  int2 c{0, 0};  // early, late
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e < own) {
      const int one = (keys[e] > border) | (keys[e] == border) << 16;
      if (e < split) c.x += one;
      else c.y += one;
    }
  int2 upto = c;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto.x, o), y = __shfl_up_sync(0xffffffffu, upto.y, o);
    if (lane >= o) upto.x += x, upto.y += y;
  }
  if (lane == 31) warp_counts[warp] = upto;
  __syncthreads();
  if (warp == 0) {
    const int2 mine = warp_counts[lane];
    int2 sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum.x, o), y = __shfl_up_sync(0xffffffffu, sum.y, o);
      if (lane >= o) sum.x += x, sum.y += y;
    }
    warp_counts[lane] = make_int2(sum.x - mine.x, sum.y - mine.y);
    if (lane == 31) cta_counts = {sum.x & 0xFFFF, sum.x >> 16, sum.y & 0xFFFF, sum.y >> 16};
  }
  cluster.sync();
  Counts cta{0, 0, 0, 0};  // before this CTA
#pragma unroll
  for (int r = 0; r < kMaxCluster; ++r)
    if (r < rank) cta = cta + *cluster.map_shared_rank(&cta_counts, r);
  cluster_arrive();  // this CTA's reads of the others are done; they may leave after cluster_wait
  const int2 in_cta = make_int2(upto.x - c.x + warp_counts[warp].x, upto.y - c.y + warp_counts[warp].y);
  const Counts before = cta + Counts{in_cta.x & 0xFFFF, in_cta.x >> 16, in_cta.y & 0xFFFF, in_cta.y >> 16};

  // Places to fill and to move before a point: of the equal keys the first `want` are kept, the early
  // ones first.
  const auto holes_before = [&](const Counts& n, int place) {
    return min(place, a.keep) - n.above_early - min(n.equal_early, want);
  };
  const auto movers_before = [&](const Counts& n) {
    return n.above_late + min(n.equal_early + n.equal_late, want) - min(n.equal_early, want);
  };
  const int holes0 = holes_before(cta, cta_first), movers0 = movers_before(cta);
  const Counts ends = cta + cta_counts;
  const int n_holes = holes_before(ends, cta_last) - holes0, n_movers = movers_before(ends) - movers0;
  // the CTA's holes from the start of the buffer, its movers from its end downwards: together they are
  // no more than its places
  int* listed = reinterpret_cast<int*>(dynamic);
  constexpr int kEnd = kThreads * E - 1;
  int equals = before.equal_early + before.equal_late;
  int hole = holes_before(before, first) - holes0, late = movers_before(before) - movers0;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e < own) {
      const bool equal = keys[e] == border;
      const bool kept = keys[e] > border || (equal && equals < want);
      equals += equal;
      if (e < split) {
        if (!kept) listed[hole++] = first + e;
      } else if (kept) {
        listed[kEnd - late++] = first + e;
      }
    }
  __syncthreads();
  int32_t* holes = a.holes + static_cast<long long>(list) * a.keep + holes0;
  int32_t* movers = a.movers + static_cast<long long>(list) * (a.n - a.keep) + movers0;
  for (int i = threadIdx.x; i < n_holes; i += kThreads) holes[i] = listed[i];
  for (int i = threadIdx.x; i < n_movers; i += kThreads) movers[i] = listed[kEnd - i];
  if (rank == ranks - 1) {
    if (threadIdx.x == 0) a.counts[list] = movers0 + n_movers;  // behind the last place: all movers
    if (list == 0) write_valid_counts(a);
  }
  cluster_wait();
}

// Pool row (in tokens) of a place, or -1 for a refused block.
__device__ __forceinline__ long long token_row(const EvictArgs& a, int place, Divisor bt) {
  const int slot = divide(place, bt);
  const int blk = a.table ? a.table[slot] : slot;
  if (blk < 0 || blk >= a.n_pool) return -1;
  return static_cast<long long>(blk) * a.bt + (place - slot * a.bt);
}

// 2^lanes_log2 lanes take a moved row of one KV head: a unit of codes (U) of K or V a lane, a unit of
// scales (S) of K or V on the first ones, its weight and position on the first two; kRows rows are in
// flight a lane. For rows of up to 16 units of K and pools of less than 2^31 token rows.
template <typename U, typename S>
__global__ void __launch_bounds__(256, 4) evict_move_kernel(const EvictArgs a, int code_units,
                                                         int scale_units, int lanes_log2, Divisor bt) {
  constexpr int kRows = 2;
  // neighbouring CTAs take the same rows of different heads, which lie next to each other
  const int list = blockIdx.x % a.kvh, l = threadIdx.x & ((1 << lanes_log2) - 1), per_cta = 256 >> lanes_log2;
  const bool has_code = l < 2 * code_units, has_scale = l < 2 * scale_units;
  U* codes = reinterpret_cast<U*>(a.packed[l >= code_units]) + list * code_units + l - (l >= code_units ? code_units : 0);
  S* scales = reinterpret_cast<S*>(a.scales[l >= scale_units]) + list * scale_units + l - (l >= scale_units ? scale_units : 0);
  const int code_step = a.kvh * code_units, scale_step = a.kvh * scale_units;
  const int32_t* stat_from = l == 0 ? reinterpret_cast<const int32_t*>(a.weights) + list * a.weights_stride
                                    : a.positions + list * a.positions_stride;
  int32_t* stat_to = (l == 0 ? reinterpret_cast<int32_t*>(a.new_weights) : a.new_positions) +
                     static_cast<long long>(list) * a.columns;
  pdl_wait();
  pdl_launch();
  const int32_t* holes = a.holes + static_cast<long long>(list) * a.keep;
  const int32_t* movers = a.movers + static_cast<long long>(list) * (a.n - a.keep);
  const int count = a.counts[list], step = gridDim.x / a.kvh * per_cta;
  if (count == 0) return;
  int from_place[kRows], to_place[kRows];
  const auto look_up = [&](int j0) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int j = min(j0 + i * step, count - 1);  // the last row again: the same bytes
      from_place[i] = movers[j];
      to_place[i] = holes[j];
    }
  };
  int j0 = blockIdx.x / a.kvh * per_cta + (threadIdx.x >> lanes_log2);
  look_up(j0);
  for (; j0 < count; j0 += kRows * step) {
    int from[kRows], to[kRows], from_stat[kRows], to_stat[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      from[i] = static_cast<int>(token_row(a, from_place[i], bt));
      to[i] = static_cast<int>(token_row(a, to_place[i], bt));
      if (from[i] < 0) to[i] = -1;
      from_stat[i] = from_place[i], to_stat[i] = to_place[i];
    }
    look_up(j0 + kRows * step);  // of the next rows, while these move
    U code[kRows];
    S scale[kRows];
    int32_t stat[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (has_code && to[i] >= 0) code[i] = codes[static_cast<long long>(from[i]) * code_step];
      if (has_scale && to[i] >= 0) scale[i] = scales[static_cast<long long>(from[i]) * scale_step];
      if (l < 2) stat[i] = stat_from[from_stat[i]];
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (has_code && to[i] >= 0) codes[static_cast<long long>(to[i]) * code_step] = code[i];
      if (has_scale && to[i] >= 0) scales[static_cast<long long>(to[i]) * scale_step] = scale[i];
      if (l < 2) stat_to[to_stat[i]] = stat[i];
    }
  }
}

// Any other row: 32 lanes take one. With one choice for all heads a row is a whole token (its heads are
// contiguous) and has the statistics of every head.
template <typename U, typename S>
__global__ void __launch_bounds__(256) evict_move_rows_kernel(const EvictArgs a, int code_units,
                                                              int scale_units, Divisor bt) {
  const int list = blockIdx.y, heads = a.shared ? 1 : a.kvh, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch();
  const int32_t* holes = a.holes + static_cast<long long>(list) * a.keep;
  const int32_t* movers = a.movers + static_cast<long long>(list) * (a.n - a.keep);
  const int count = a.counts[list];
  for (int j = blockIdx.x * 8 + (threadIdx.x >> 5); j < count; j += gridDim.x * 8) {
    const int from_place = movers[j], to_place = holes[j];
    const long long from = token_row(a, from_place, bt), to = token_row(a, to_place, bt);
    if (from >= 0 && to >= 0)
      for (int kv = 0; kv < 2; ++kv) {
        U* codes = reinterpret_cast<U*>(a.packed[kv]);
        S* scales = reinterpret_cast<S*>(a.scales[kv]);
        for (int u = lane; u < code_units; u += 32)
          codes[(to * heads + list) * code_units + u] = codes[(from * heads + list) * code_units + u];
        for (int u = lane; u < scale_units; u += 32)
          scales[(to * heads + list) * scale_units + u] = scales[(from * heads + list) * scale_units + u];
      }
    for (int h = list + lane; h < (a.shared ? a.kvh : list + 1); h += 32) {
      const long long row = static_cast<long long>(h) * a.columns;
      a.new_weights[row + to_place] = a.weights[h * a.weights_stride + from_place];
      a.new_positions[row + to_place] = a.positions[h * a.positions_stride + from_place];
    }
  }
}

template <typename U, typename S>
cudaError_t move_as(const EvictArgs& a, int code_bytes, int scale_bytes, cudaStream_t s) {
  const int lists = a.shared ? 1 : a.kvh;
  const int codes = code_bytes / static_cast<int>(sizeof(U)), scales = scale_bytes / static_cast<int>(sizeof(S));
  int log2 = 0;
  while (log2 < 5 && (1 << log2) < 2 * codes) ++log2;
  const Divisor bt = divisor(static_cast<unsigned>(a.bt));
  if (!a.shared && codes <= 16 && 2 * scales <= 1 << log2 && static_cast<long long>(a.n_pool) * a.bt <= 0x7fffffff)
    return launch_pdl(evict_move_kernel<U, S>, dim3((148 * 4 + a.kvh - 1) / a.kvh * a.kvh), 256, 0, s, a, codes,
                      scales, log2, bt);
  return launch_pdl(evict_move_rows_kernel<U, S>, dim3((148 * 8 + lists - 1) / lists, lists), 256, 0, s, a, codes, scales, bt);
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

namespace {

// Launches kernel(args...) as clusters of `ranks` CTAs, one per choice.
template <typename... Params, typename... Given>
cudaError_t launch_select(void (*kernel)(Params...), int ranks, int lists, size_t smem, cudaStream_t s,
                          Given... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranks, lists, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ranks;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

template <int E>
cudaError_t select_in_registers(const EvictArgs& a, int ranks, int lists, int vectors, cudaStream_t s) {
  const auto kernel = evict_select_kernel<E>;
  constexpr size_t smem = sizeof(unsigned) * (kThreads * E + 2 * kDigits);
  if (smem >= 48 * 1024) {  // with the kernel's static shared memory more than is had unasked
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
  }
  const int run = ((a.n + ranks - 1) / ranks + 3) / 4 * 4;  // vectors of 4 places stay whole
  return launch_select(kernel, ranks, lists, smem, s, a, run, vectors);
}

cudaError_t select(const EvictArgs& a, int lists, cudaStream_t s) {
  // As many CTAs a choice as the SMs give room for, from 4096 places a CTA on (10007 places, one choice:
  // 4 CTAs 20.7 us, 8 CTAs 25.9 us, whose barriers and remote reads cost more than they share).
  int ranks = 1;
  while (ranks < kMaxCluster && 2 * ranks * lists <= 148 && a.n > ranks * kThreads * 4) ranks *= 2;
  while (ranks < kMaxCluster && a.n > ranks * kThreads * 16) ranks *= 2;  // or as its places need
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.weights) | reinterpret_cast<uintptr_t>(a.positions) |
                       reinterpret_cast<uintptr_t>(a.new_weights) | reinterpret_cast<uintptr_t>(a.new_positions);
  const int vectors = at % 16 == 0 && (a.weights_stride | a.positions_stride | a.columns) % 4 == 0;
  if (a.n <= ranks * kThreads * 4) return select_in_registers<4>(a, ranks, lists, vectors, s);
  if (a.n <= ranks * kThreads * 8) return select_in_registers<8>(a, ranks, lists, vectors, s);
  if (a.n <= ranks * kThreads * 16) return select_in_registers<16>(a, ranks, lists, vectors, s);
  const int run = static_cast<int>((static_cast<long long>(a.n) + kLongCluster * 32 - 1) / (kLongCluster * 32) * 32);
  const int cached = run <= kMaxCached;  // evict_scratch_ints has room for the keys otherwise
  const cudaError_t e = cudaFuncSetAttribute(evict_select_long_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             kMaxCached * sizeof(unsigned));
  if (e != cudaSuccess) return e;
  return launch_select(evict_select_long_kernel, kLongCluster, lists, cached ? run * sizeof(unsigned) : 0, s, a,
                       run, cached, vectors);
}

}  // namespace

size_t evict_scratch_ints(int n, int lists) {
  const size_t listed = static_cast<size_t>(lists) * (static_cast<size_t>(n) + 1);
  return n > kLongCluster * (kMaxCached - 32) ? listed + static_cast<size_t>(lists) * n : listed;
}

cudaError_t launch_evict(const EvictArgs& a, cudaStream_t s) {
  const int lists = a.shared ? 1 : a.kvh;
  const cudaError_t e = select(a, lists, s);
  if (e != cudaSuccess) return e;
  const int heads = a.shared ? a.kvh : 1;
  const int code_bytes = heads * a.packed_dim, scale_bytes = heads * a.groups * 2;
  const uintptr_t cp = reinterpret_cast<uintptr_t>(a.packed[0]) | reinterpret_cast<uintptr_t>(a.packed[1]) | code_bytes;
  if (cp % 16 == 0) return move_codes<uint4>(a, code_bytes, scale_bytes, s);
  if (cp % 4 == 0) return move_codes<uint32_t>(a, code_bytes, scale_bytes, s);
  return move_codes<uint8_t>(a, code_bytes, scale_bytes, s);
}

}  // namespace kvb
