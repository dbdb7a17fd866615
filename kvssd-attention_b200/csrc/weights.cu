// Attention weights over the packed keys: for each KV head and each selected place
//   out = previous + sum over the queries and the query heads of that KV head of exp(s - lse),
//   s = sm_scale * sum_d q_d * (code_d - 2^(bits-1)) * scale,
// zero where the query does not see the place (rows behind valid_tokens, places from the query's
// `visible` count on, refused blocks). The log-sum-exps come from the attention that has run, or a
// first pass over the keys computes them.
//
// head_dim 64, 96, 128 and 256 with scale groups of whole 16 dims and aligned codes run on the
// tensor cores: up to 8 query rows a KV head by weights_step.cuh, up to 32 by weights_window.cuh, more by
// weights_umma.cuh. weights_lse_kernel, weights_combine_kernel and weights_kernel are the
// form for any other shape: a CTA takes one KV head and kPlaces places, a warp one place at a time,
// the lanes the head's dims.
#include "weights_umma.cuh"

namespace kvb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kPlaces = 32;
constexpr int kMaxPerLane = 8;  // dims of a head a lane holds (head_dim <= 256)

// The dequantized key of one (place, KV head): dims lane, lane + 32, ... Returns false where the
// place holds no valid token.
__device__ __forceinline__ bool load_key(const WeightsArgs& a, int place, int h, int lane,
                                         float (&k)[kMaxPerLane]) {
  const int slot = place / a.bt, row = place - slot * a.bt;
  const int blk = a.table ? a.table[slot] : slot;
  if (blk < 0 || blk >= a.n_pool) {
    if (a.status && lane == 0) atomicOr(a.status, kDevBadBlockIndex);
    return false;
  }
  const int valid = a.valid[blk];
  if ((valid < 0 || valid > a.bt) && a.status && lane == 0) atomicOr(a.status, kDevBadValidCount);
  if (row >= valid) return false;
  const long long r = (static_cast<long long>(blk) * a.bt + row) * a.kvh + h;
  const int per = 8 / a.bits, mid = 1 << (a.bits - 1);
  const uint8_t* codes = a.kp + r * (a.d / per);
  const __half* scales = a.ks + r * (a.d / a.group);
#pragma unroll
  for (int i = 0; i < kMaxPerLane; ++i) {
    const int d = lane + 32 * i;
    k[i] = 0.f;
    if (d < a.d) {
      const int code = (codes[d / per] >> (d % per * a.bits)) & ((1 << a.bits) - 1);
      k[i] = static_cast<float>(code - mid) * __half2float(scales[d / a.group]);
    }
  }
  return true;
}

__device__ __forceinline__ float score(const WeightsArgs& a, int t, int head, int lane,
                                       const float (&k)[kMaxPerLane]) {
  const long long q = (static_cast<long long>(t) * a.qh + head) * a.d;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxPerLane; ++i) {
    const int d = lane + 32 * i;
    if (d < a.d) s = fmaf(load_query(a.query, a.dtype, q + d), k[i], s);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s * a.sm_scale;
}

__device__ __forceinline__ bool sees(const WeightsArgs& a, int t, int place) {
  return !a.visible || place < a.visible[t];
}

// (m, l) joined with another such part. One that has seen nothing has l = 0; a NaN in l stays.
__device__ __forceinline__ void join(float& m, float& l, float m2, float l2) {
  if (l2 == 0.f) return;
  const float top = max(m, m2);
  l = (l == 0.f ? 0.f : l * expf(m - top)) + l2 * expf(m2 - top);
  m = top;
}

// Parts (m, l) of each query row: scratch [parts][rows][2]. A CTA takes the run of kPlaces places of its
// number or, RUNS, every gridDim.x-th one from it on, and joins what it finds with what it has found before.
template <bool RUNS>
__global__ void __launch_bounds__(kThreads) weights_lse_kernel(const WeightsArgs a, int chunks) {
  __shared__ float keys[kPlaces][kMaxPerLane * 32];
  __shared__ bool live[kPlaces];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.y, gqa = a.qh / a.kvh;
  pdl_wait();
  pdl_launch();
  for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int first = chunk * kPlaces, places = min(kPlaces, a.n_sel * a.bt - first);
    for (int p = warp; p < places; p += kWarps) {
      float k[kMaxPerLane];
      const bool ok = load_key(a, first + p, h, lane, k);
      if (lane == 0) live[p] = ok;
      if (ok)
        for (int i = 0; i < kMaxPerLane; ++i) keys[p][lane + 32 * i] = k[i];
    }
    __syncthreads();
    for (int r = warp; r < a.queries * gqa; r += kWarps) {
      const int t = r / gqa, head = h * gqa + r % gqa;
      float m = -INFINITY, l = 0.f;
      for (int p = 0; p < places; ++p) {
        if (!live[p] || !sees(a, t, first + p)) continue;
        float k[kMaxPerLane];
        for (int i = 0; i < kMaxPerLane; ++i) k[i] = keys[p][lane + 32 * i];
        const float s = score(a, t, head, lane, k);
        if (s == -INFINITY) continue;
        const float top = max(m, s);  // of the numbers: a NaN score reaches l, and stays in it
        l = l * expf(m - top) + expf(s - top);
        m = top;
      }
      if (lane == 0) {
        float* part = a.scratch + 2 * (static_cast<long long>(blockIdx.x) * a.queries * a.qh +
                                       static_cast<long long>(t) * a.qh + head);
        if (RUNS && chunk >= gridDim.x) join(m, l, part[0], part[1]);
        part[0] = m;
        part[1] = l;
      }
    }
    if (!RUNS) break;
    __syncthreads();
  }
}

// One warp a query row: lse = log sum_parts l e^m (-inf where the row sees nothing).
__global__ void __launch_bounds__(kThreads) weights_combine_kernel(const WeightsArgs a, int parts) {
  const int lane = threadIdx.x & 31;
  const int rows = a.queries * a.qh, row = blockIdx.x * kWarps + (threadIdx.x >> 5);
  pdl_wait();
  pdl_launch();
  if (row >= rows) return;
  float m = -INFINITY, l = 0.f;
  for (int p = lane; p < parts; p += 32) {
    const float* part = a.scratch + 2 * (static_cast<long long>(p) * rows + row);
    join(m, l, part[0], part[1]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
    join(m, l, m2, l2);
  }
  if (lane == 0) a.lse[row] = l == 0.f ? -INFINITY : m + logf(l);
}

__global__ void __launch_bounds__(kThreads) weights_kernel(const WeightsArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.y, first = blockIdx.x * kPlaces, gqa = a.qh / a.kvh;
  const int places = min(kPlaces, a.n_sel * a.bt - first);
  const float* lse = a.lse_in ? a.lse_in : a.lse;
  pdl_wait();
  pdl_launch();
  for (int p = warp; p < places; p += kWarps) {
    const int place = first + p;
    float k[kMaxPerLane], sum = 0.f;
    if (load_key(a, place, h, lane, k))
      for (int t = 0; t < a.queries; ++t) {
        if (!sees(a, t, place)) continue;
        for (int g = 0; g < gqa; ++g) {
          const float s = score(a, t, h * gqa + g, lane, k);
          const float l = lse[static_cast<long long>(t) * a.qh + h * gqa + g];
          if (l != -INFINITY) sum += expf(s - l);
        }
      }
    if (lane == 0) {
      if (a.previous) sum += a.previous[h * a.previous_stride + place];
      a.out[h * a.out_stride + place] = sum;
    }
  }
}

}  // namespace

using TcLauncher = cudaError_t (*)(const WeightsArgs&, cudaStream_t);

TcLauncher tc_launcher(int d, int group) {
  if (group % 16) return nullptr;
  switch (d) {
    case 64: return launch_weights_tc_64;
    case 96: return launch_weights_tc_96;
    case 128: return launch_weights_tc_128;
    case 256: return launch_weights_tc_256;
    default: return nullptr;
  }
}

// Parts of a query row in the log-sum-exp pass for any shape: one a run of places (131072 places x 8 heads of
// 80: 1.68 ms; as many as are resident at once, each of several runs, 1.83 ms) up to 8 MB of them in all, or
// as many as are resident.
long long general_parts(int queries, int qh, int kvh, int n_sel, int bt) {
  const long long chunks = (static_cast<long long>(n_sel) * bt + kPlaces - 1) / kPlaces;
  long long most = (1ll << 20) / (static_cast<long long>(queries) * qh);
  if (most < 148 * 4 / kvh) most = 148 * 4 / kvh;
  if (most < 1) most = 1;
  return most < chunks ? most : chunks;
}

size_t weights_scratch_bytes(int queries, int qh, int kvh, int n_sel, int bt, int d, int group) {
  long long parts = general_parts(queries, qh, kvh, n_sel, bt);  // of any shape off 16 bytes too
  if (tc_launcher(d, group)) {
    const int tiles = n_sel * ((bt + 15) / 16);  // of the narrower windows, at most
    const int window = weights_tc::grid_x(tiles, kvh, 1, weights_tc::kWarps, 2);
    parts = window > parts ? window : parts;
    for (int ctas = 1; ctas <= 2; ++ctas) {  // an SM, by the shape and the queries' type
      const int wide = weights_umma::plan(n_sel, bt, kvh, ctas).parts;
      parts = wide > parts ? wide : parts;
    }
  }
  return static_cast<size_t>(parts) * queries * qh * 2 * sizeof(float);
}

cudaError_t launch_weights(const WeightsArgs& a, cudaStream_t s) {
  const TcLauncher tc = tc_launcher(a.d, a.group);
  if (tc && (reinterpret_cast<uintptr_t>(a.kp) | reinterpret_cast<uintptr_t>(a.ks)) % 16 == 0)
    return tc(a, s);
  const int chunks = (a.n_sel * a.bt + kPlaces - 1) / kPlaces;
  if (!a.lse_in) {
    const int parts = static_cast<int>(general_parts(a.queries, a.qh, a.kvh, a.n_sel, a.bt));
    if (parts > a.parts_room) return cudaErrorInvalidValue;
    cudaError_t e = launch_pdl(parts < chunks ? weights_lse_kernel<true> : weights_lse_kernel<false>,
                               dim3(parts, a.kvh), kThreads, 0, s, a, chunks);
    if (e != cudaSuccess) return e;
    e = launch_pdl(weights_combine_kernel, dim3((a.queries * a.qh + kWarps - 1) / kWarps), kThreads,
                   0, s, a, parts);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(weights_kernel, dim3(chunks, a.kvh), kThreads, 0, s, a);
}

}  // namespace kvb
