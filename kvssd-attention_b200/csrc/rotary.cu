// Rotary positions: of each head's first 2 * pairs dims, pair i = (a, b) becomes
//   m * (a cos t - b sin t),  m * (b cos t + a sin t),   t = position * frequency_i,
// with b = dim i + pairs (half layout) or the pairs interleaved (dims 2i, 2i + 1); the dims behind
// are copied. Bound by HBM: every element is read and written once, at 3 flops.
//
// The angle is taken in FP64 and reduced to a fraction of a turn there (at a position of 10^6 an
// FP32 angle is off by 0.03 rad); cos and sin of the reduced angle, the products and their sum are
// FP32, rounded once to the element type.
#include "cache_ops.cuh"

namespace kvb {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 4;  // items a thread has in flight

// cos and sin (times the magnitude) of one (token, pair).
__device__ __forceinline__ float2 cos_sin(const RotaryArgs& a, int token, int pair) {
  const double f = turn_fraction(index_at(a.positions, token), a.freq[pair]);
  float s, c;
  sincospif(static_cast<float>(2.0 * f), &s, &c);
  return make_float2(c * a.magnitude, s * a.magnitude);
}

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

// An item is V pairs of one (token, head) row -- two vectors of V elements: dims [V j, V j + V) and
// the same plus `pairs` (half layout), or the 2 V dims from 2 V j on (interleaved) -- or, behind the
// rotated part, up to 2 V dims to copy. A CTA takes `span` whole tokens: it first fills a table of
// their cos and sin in shared memory (each used by all heads), while the first items' loads are in
// flight, then works through the items, kBatch per thread at a time so that 128 bytes a thread are
// in flight with 16-byte vectors.
template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a, int span, int chunks) {
  extern __shared__ float2 table[];  // [span][pairs]
  const int first = blockIdx.x * span;
  const int tokens = min(span, a.tokens - first);
  const int per_token = a.heads * chunks;
  const int items = tokens * per_token;
  const int rotated = a.pairs / V;
  const T* x = static_cast<const T*>(a.x.p);
  T* out = static_cast<T*>(a.out);
  using VecT = Vec<T, V>;

  pdl_wait();
  pdl_launch();
  bool filled = false;
  for (int base = 0; base < items; base += kThreads * kBatch) {
    VecT lo[kBatch], hi[kBatch];
    int tok[kBatch], chunk[kBatch];
    long long to[kBatch];
    bool two[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int item = base + u * kThreads + static_cast<int>(threadIdx.x);
      tok[u] = -1;
      if (item < items) {
        const int t = item / per_token, rest = item - t * per_token;
        const int h = rest / chunks, c = rest - h * chunks;
        tok[u] = t;
        chunk[u] = c;
        const int d0 = c < rotated && !kInterleaved ? c * V : 2 * c * V;
        const int d1 = c < rotated && !kInterleaved ? d0 + a.pairs : d0 + V;
        two[u] = d1 < a.d;
        const T* src = x + (first + t) * a.x.token + h * a.x.head;
        to[u] = (first + t) * a.out_token + h * a.out_head;
        lo[u] = *reinterpret_cast<const VecT*>(src + d0);
        if (two[u]) hi[u] = *reinterpret_cast<const VecT*>(src + d1);
      }
    }
    if (!filled) {
      filled = true;
      for (int i = threadIdx.x; i < tokens * a.pairs; i += kThreads) {
        const int t = i / a.pairs;
        table[i] = cos_sin(a, first + t, i - t * a.pairs);
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (tok[u] < 0) continue;
      const int c = chunk[u];
      const int d0 = c < rotated && !kInterleaved ? c * V : 2 * c * V;
      const int d1 = c < rotated && !kInterleaved ? d0 + a.pairs : d0 + V;
      if (c < rotated) {
        const float2* cs = table + tok[u] * a.pairs + c * V;
        if constexpr (kInterleaved) {
#pragma unroll
          for (int i = 0; i < V; ++i) {  // pair i of the item: elements 2i, 2i + 1 of (lo, hi)
            T& ea = 2 * i < V ? lo[u].e[2 * i % V] : hi[u].e[2 * i % V];
            T& eb = 2 * i + 1 < V ? lo[u].e[(2 * i + 1) % V] : hi[u].e[(2 * i + 1) % V];
            const float p = to_f32(ea), q = to_f32(eb);
            ea = from_f32<T>(p * cs[i].x - q * cs[i].y);
            eb = from_f32<T>(q * cs[i].x + p * cs[i].y);
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float p = to_f32(lo[u].e[i]), q = to_f32(hi[u].e[i]);
            lo[u].e[i] = from_f32<T>(p * cs[i].x - q * cs[i].y);
            hi[u].e[i] = from_f32<T>(q * cs[i].x + p * cs[i].y);
          }
        }
      }
      *reinterpret_cast<VecT*>(out + to[u] + d0) = lo[u];
      if (two[u]) *reinterpret_cast<VecT*>(out + to[u] + d1) = hi[u];
    }
  }
}

template <typename T, int V>
cudaError_t launch(const RotaryArgs& a, cudaStream_t s) {
  const int chunks = a.pairs / V + (a.d - 2 * a.pairs + 2 * V - 1) / (2 * V);
  const long long per_token = static_cast<long long>(a.heads) * chunks;
  // As many tokens a CTA as give each thread a full batch, but no more than the GPU's threads
  // share out when there are few (one item a thread has the least latency then), and no more than
  // 32 KB of table.
  long long span = kThreads * kBatch / per_token;
  const long long few = (static_cast<long long>(a.tokens) + 295) / 296;
  if (span > few) span = few;
  const long long room = a.pairs ? 32768 / (8 * a.pairs) : a.tokens;
  if (span > room) span = room;
  if (span < 1) span = 1;
  const unsigned grid = static_cast<unsigned>((a.tokens + span - 1) / span);
  const size_t smem = static_cast<size_t>(span) * a.pairs * sizeof(float2);
  auto kernel = a.interleaved ? rotary_kernel<T, V, true> : rotary_kernel<T, V, false>;
  return launch_pdl(kernel, dim3(grid), kThreads, smem, s, a, static_cast<int>(span), chunks);
}

template <typename T>
cudaError_t dispatch(const RotaryArgs& a, cudaStream_t s) {
  // 16-byte vectors where every row and both vectors of an item start on 16 bytes; else by element.
  constexpr int V = 16 / sizeof(T);
  const long long rows = a.x.token | a.x.head | a.out_token | a.out_head;
  const bool aligned = ((reinterpret_cast<uintptr_t>(a.x.p) | reinterpret_cast<uintptr_t>(a.out)) & 15) == 0;
  if (aligned && rows % V == 0 && a.pairs % V == 0 && a.d % V == 0) return launch<T, V>(a, s);
  return launch<T, 1>(a, s);
}

}  // namespace

cudaError_t launch_rotary(const RotaryArgs& a, cudaStream_t s) {
  switch (a.dtype) {
    case kQF16: return dispatch<__half>(a, s);
    case kQBF16: return dispatch<__nv_bfloat16>(a, s);
    default: return dispatch<float>(a, s);
  }
}

}  // namespace kvb
