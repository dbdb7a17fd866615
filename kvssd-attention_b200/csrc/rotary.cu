// Rotary positions: of each head's first 2 * pairs dims, pair i = (a, b) becomes
//   m * (a cos t - b sin t),  m * (b cos t + a sin t),   t = position * frequency_i,
// with b = dim i + pairs (half layout) or the pairs interleaved (dims 2i, 2i + 1); the dims behind
// are copied. Bound by HBM: every element is read and written once, at 3 flops.
//
// The angle is taken in FP64 and reduced to a fraction of a turn there (at a position of 10^6 an
// FP32 angle is off by 0.03 rad); cos and sin of the reduced angle, the products and their sum are
// FP32, rounded once to the element type.
//
// 8192 x 32 x 128 BF16: 22.7 us, 5.9 TB/s (0.90 of the measured copy rate), two batches a thread; with one
// 24.0 us. With arrays of 16-bit elements in place of 32-bit words it took 40.6 us, and with divisions
// in the loop 49.5.
#include "cache_ops.cuh"

namespace kvb {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 2;     // items a thread has in flight
constexpr int kResident = 4;  // CTAs on an SM

// cos and sin (times the magnitude) of one (token, pair).
__device__ __forceinline__ float2 cos_sin(const RotaryArgs& a, int token, int pair) {
  const double f = turn_fraction(index_at(a.positions, token), a.freq[pair]);
  float s, c;
  sincospif(static_cast<float>(2.0 * f), &s, &c);
  return make_float2(c * a.magnitude, s * a.magnitude);
}

// V elements: one, or the words of 16 bytes.
template <typename T, int V>
struct alignas(16) Vec {
  uint32_t w[4];
  __device__ __forceinline__ void load(const T* p) {
    *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
  }
  __device__ __forceinline__ void store(T* p) const {
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(w);
  }
};
template <typename T>
struct Vec<T, 1> {
  T e;
  __device__ __forceinline__ void load(const T* p) { e = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = e; }
};

// An item is V pairs of one (token, head) row -- two vectors of V elements: dims [V j, V j + V) and
// the same plus `pairs` (half layout), or the 2 V dims from 2 V j on (interleaved) -- or, behind the
// rotated part, up to 2 V dims to copy. A CTA takes `span` whole tokens. Each thread keeps to one of a
// row's items (so nothing is divided in the loop) and walks over the rows, kBatch of them in flight. The
// tokens' cos and sin are put into shared memory first, while the
// first items load, and used by all heads: entry [token][i][j] for pair i of item j, so that a warp
// reads neighbouring entries.
template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, kResident) rotary_kernel(const RotaryArgs a, int span, int chunks) {
  extern __shared__ float2 table[];
  const int first = blockIdx.x * span;
  const int tokens = min(span, a.tokens - first);
  const int rotated = a.pairs / V;                   // items of a row that turn
  const int step = kThreads / chunks;                // rows the CTA's threads take at a time
  const int c = threadIdx.x % chunks, lane_row = threadIdx.x / chunks;
  const bool halves = c < rotated && !kInterleaved;
  const int d0 = halves ? c * V : 2 * c * V, d1 = halves ? d0 + a.pairs : d0 + V;
  const bool two = d1 < a.d;
  const int token_stride = static_cast<int>(a.x.token), head_stride = static_cast<int>(a.x.head);
  const int out_token = static_cast<int>(a.out_token), out_head = static_cast<int>(a.out_head);
  const T* x = static_cast<const T*>(a.x.p) + first * a.x.token + d0;
  T* out = static_cast<T*>(a.out) + first * a.out_token + d0;
  const int apart = d1 - d0;
  const int step_tokens = step / a.heads, step_heads = step - step_tokens * a.heads;
  int t = lane_row / a.heads, h = lane_row - t * a.heads;  // the thread's next row
  if (lane_row >= step) t = tokens;                        // threads left over
  using VecT = Vec<T, V>;

  pdl_wait();
  pdl_launch();
  bool filled = false;
  do {
    VecT lo[kBatch], hi[kBatch];
    int tok[kBatch];
    T* to[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      tok[u] = t;
      if (t < tokens) {
        const T* src = x + (static_cast<long long>(t) * token_stride + static_cast<long long>(h) * head_stride);
        to[u] = out + (static_cast<long long>(t) * out_token + static_cast<long long>(h) * out_head);
        lo[u].load(src);
        if (two) hi[u].load(src + apart);
      }
      t += step_tokens;
      h += step_heads;
      if (h >= a.heads) h -= a.heads, ++t;
    }
    if (!filled) {
      filled = true;
      for (int i = threadIdx.x; i < tokens * a.pairs; i += kThreads) {
        const int token = i / a.pairs, pair = i - token * a.pairs;
        table[token * a.pairs + pair % V * rotated + pair / V] = cos_sin(a, first + token, pair);
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (tok[u] >= tokens) continue;
      if (c < rotated) {
        const float2* cs = table + tok[u] * a.pairs + c;
        if constexpr (V == 1) {
          const float2 turn = cs[0];
          const float p = to_f32(lo[u].e), q = to_f32(hi[u].e);
          lo[u].e = from_f32<T>(__fmaf_rn(q, -turn.y, __fmul_rn(p, turn.x)));
          hi[u].e = from_f32<T>(__fmaf_rn(p, turn.y, __fmul_rn(q, turn.x)));
        } else if constexpr (kInterleaved) {
#pragma unroll
          for (int i = 0; i < V; ++i) {  // pair i of the item: one of lo, then one of hi
            uint32_t* w = i < V / 2 ? lo[u].w : hi[u].w;
            const int at = i % (V / 2);
            const float2 turn = cs[i * rotated];
            const F2 p = unpack_pair<T>(w, at);
            const float2 two_of = parts(p);
            pack_pair<T>(fma2(f2(two_of.y, two_of.x), f2(-turn.y, turn.y), mul2(p, f2(turn.x))), w, at);
          }
        } else {
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {  // two pairs an instruction
            const float2 t0 = cs[2 * i * rotated], t1 = cs[(2 * i + 1) * rotated];
            const F2 cos = f2(t0.x, t1.x), sin = f2(t0.y, t1.y), minus = f2(-t0.y, -t1.y);
            const F2 p = unpack_pair<T>(lo[u].w, i), q = unpack_pair<T>(hi[u].w, i);
            pack_pair<T>(fma2(q, minus, mul2(p, cos)), lo[u].w, i);
            pack_pair<T>(fma2(p, sin, mul2(q, cos)), hi[u].w, i);
          }
        }
      }
      lo[u].store(to[u]);
      if (two) hi[u].store(to[u] + apart);
    }
  } while (t < tokens);
}

template <typename T, int V>
cudaError_t launch(const RotaryArgs& a, cudaStream_t s) {
  const int chunks = a.pairs / V + (a.d - 2 * a.pairs + 2 * V - 1) / (2 * V);
  const int rows = kThreads / chunks;  // at a time
  // As many tokens a CTA as give each thread two batches (8192 x 32 x 128 BF16: 22.7 us, one batch 24.0),
  // but no more than spread few tokens over the GPU (one item a thread has the least latency then), and
  // no more than 32 KB of table.
  long long span = static_cast<long long>(rows) * kBatch * 2 / a.heads;
  const long long few = (static_cast<long long>(a.tokens) + 295) / 296;
  if (span > few) span = few;
  const long long room = 32768 / (8 * a.pairs);
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
