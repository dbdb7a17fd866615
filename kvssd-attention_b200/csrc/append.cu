// The quantizing cache write: each token's keys (rotated first where frequencies are given) and
// values become groupwise INT2/INT4 codes and FP16 scales in the token's slot of the block pool, in
// the layout of kvssd's quantizer (src/kvssd/quant.py:28-65):
//   scale = max|x| / (2^(bits-1) - 1) in FP32, at least 1e-8 / (...); code = round-half-even(x / scale)
//   + 2^(bits-1); codes packed low bits first; the scale stored as FP16.
// Scale and quotient are the correctly rounded FP32 divisions, so the codes are those of the
// quantizer bit for bit. Rotated keys are computed as a pair of FP32 numbers (cos and sin as pairs,
// products and sum with their rounding errors) and rounded to FP32 once, so that the codes do not
// depend on the order of roundings; they are not rounded to the input's type in between.
//
// Bound by HBM: the inputs are read once, codes and scales (and, when asked for, the FP16 values
// that the codes stand for) are written once.
//
// append_kernel is the form for any shape and alignment: a CTA takes one token, a warp one scale
// group after the other, a lane one byte of codes after the other.
#include "cache_ops.cuh"

namespace kvb {
namespace {

constexpr int kThreads = 256;

// (hi, lo) pairs of m cos t and m sin t.
struct Turn {
  float ch, cl, sh, sl;
};

__device__ __forceinline__ Turn make_turn(long long position, double freq, float magnitude) {
  double s, c;
  sincospi(2.0 * turn_fraction(position, freq), &s, &c);
  c *= static_cast<double>(magnitude);
  s *= static_cast<double>(magnitude);
  Turn t;
  t.ch = static_cast<float>(c);
  t.cl = static_cast<float>(c - static_cast<double>(t.ch));
  t.sh = static_cast<float>(s);
  t.sl = static_cast<float>(s - static_cast<double>(t.sh));
  return t;
}

// x c + y s rounded once: products and sum with their rounding errors (Dekker, Knuth), to about
// 2^-45 of the larger product before the last rounding.
__device__ __forceinline__ float rotate_once(float x, float y, const Turn& t, float sign) {
  const float sh = sign * t.sh, sl = sign * t.sl;
  const float p = __fmul_rn(x, t.ch), pe = __fmaf_rn(x, t.ch, -p);
  const float q = __fmul_rn(y, sh), qe = __fmaf_rn(y, sh, -q);
  const float sum = __fadd_rn(p, q);
  const float b = __fsub_rn(sum, p);
  const float e = __fadd_rn(__fsub_rn(p, __fsub_rn(sum, b)), __fsub_rn(q, b));
  const float low = __fmaf_rn(x, t.cl, __fmaf_rn(y, sl, __fadd_rn(pe, qe)));
  return __fadd_rn(sum, __fadd_rn(low, e));
}

// max that keeps a NaN, so that a group with a NaN gets a NaN scale.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The pool row of `slot`, or -1 (a negative slot: padding; one behind the pool: refused, flagged).
__device__ __forceinline__ long long pool_row(const AppendArgs& a, long long slot) {
  if (slot < 0) return -1;
  if (slot >= static_cast<long long>(a.n_pool) * a.bt) {
    if (a.status) atomicOr(a.status, kDevBadBlockIndex);
    return -1;
  }
  return slot;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs a) {
  extern __shared__ Turn turns[];  // [pairs]
  const int token = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  pdl_launch();
  const long long row = pool_row(a, index_at(a.slots, token));
  if (a.freq) {
    const long long position = index_at(a.positions, token);
    for (int i = threadIdx.x; i < a.pairs; i += kThreads)
      turns[i] = make_turn(position, a.freq[i], a.magnitude);
    __syncthreads();
  }
  if (threadIdx.x == 0 && row >= 0 && a.valid)
    atomicMax(a.valid + row / a.bt, static_cast<int>(row % a.bt) + 1);
  const int groups = a.d / a.group, per = 8 / a.bits, mid = 1 << (a.bits - 1);
  const int bytes = a.group / per;
  const int pairs = a.freq ? a.pairs : 0;
  for (int g = warp; g < 2 * a.kvh * groups; g += kThreads / 32) {
    const int kv = g / (a.kvh * groups), h = g / groups % a.kvh, gi = g % groups;
    const RowTensor& in = kv ? a.value : a.key;
    const T* x = static_cast<const T*>(in.p) + token * in.token + h * in.head;
    const auto element = [&](int d) -> float {
      const float own = to_f32(x[d]);
      if (kv || d >= 2 * pairs) return own;
      const int pair = a.interleaved ? d >> 1 : (d < pairs ? d : d - pairs);
      const bool second = a.interleaved ? (d & 1) : d >= pairs;
      const int other = a.interleaved ? d ^ 1 : (second ? d - pairs : d + pairs);
      return rotate_once(own, to_f32(x[other]), turns[pair], second ? 1.f : -1.f);
    };
    float top = 0.f;
    for (int b = lane; b < bytes; b += 32)
      for (int i = 0; i < per; ++i)
        top = max_nan(top, fabsf(element(gi * a.group + b * per + i)));
#pragma unroll
    for (int o = 16; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float scale = __fdiv_rn(max_nan(top, 1e-8f), static_cast<float>(mid - 1));
    const __half held = __float2half_rn(scale);
    if (row >= 0 && lane == 0) a.scales[kv][(row * a.kvh + h) * groups + gi] = held;
    for (int b = lane; b < bytes; b += 32) {
      unsigned byte = 0;
      for (int i = 0; i < per; ++i) {
        const int d = gi * a.group + b * per + i;
        int n = __float2int_rn(__fdiv_rn(element(d), scale));  // NaN: 0
        n = max(-mid, min(mid - 1, n));
        byte |= static_cast<unsigned>(n + mid) << (i * a.bits);
        if (a.values[kv])
          a.values[kv][(static_cast<long long>(token) * a.kvh + h) * a.d + d] =
              __float2half_rn(static_cast<float>(n) * __half2float(held));
      }
      if (row >= 0)
        a.packed[kv][(row * a.kvh + h) * (a.d / per) + gi * bytes + b] = static_cast<uint8_t>(byte);
    }
  }
}

template <typename T>
cudaError_t dispatch(const AppendArgs& a, cudaStream_t s) {
  const size_t smem = a.freq ? a.pairs * sizeof(Turn) : 0;
  return launch_pdl(append_kernel<T>, dim3(a.tokens), kThreads, smem, s, a);
}

}  // namespace

cudaError_t launch_append(const AppendArgs& a, cudaStream_t s) {
  switch (a.dtype) {
    case kQF16: return dispatch<__half>(a, s);
    case kQBF16: return dispatch<__nv_bfloat16>(a, s);
    default: return dispatch<float>(a, s);
  }
}

}  // namespace kvb
