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
// that the codes stand for) are written once; the arithmetic of the rotated keys comes close to that
// time, so it is kept short where it can be (rotate_once, quantize8).
//
// append_rows_kernel: scale groups and pairs of whole 8 elements, rows on 16 bytes. append_kernel is
// the form for any other shape and alignment: a CTA takes one token, a warp one scale group after the
// other, a lane one byte of codes after the other.
#include "cache_ops.cuh"

namespace kvb {
namespace {

constexpr int kThreads = 256;

// (hi, lo) pairs of m cos t and m sin t.
struct Turn {
  float ch, cl, sh, sl;
};

// A 16-bit element times ch must be exact in FP32 for rotate_once: ch then has 13 bits.
template <typename T>
__device__ __forceinline__ float high_part(double x) {
  const float f = static_cast<float>(x);
  return sizeof(T) == 2 ? __uint_as_float(__float_as_uint(f) & 0xFFFFF800u) : f;
}

template <typename T>
__device__ __forceinline__ Turn make_turn(long long position, double freq, float magnitude) {
  double s, c;
  sincospi(2.0 * turn_fraction(position, freq), &s, &c);
  c *= static_cast<double>(magnitude);
  s *= static_cast<double>(magnitude);
  Turn t;
  t.ch = high_part<T>(c);
  t.cl = static_cast<float>(c - static_cast<double>(t.ch));
  t.sh = high_part<T>(s);
  t.sl = static_cast<float>(s - static_cast<double>(t.sh));
  return t;
}

// x c + y s rounded once: the rounding errors of the products (none for a 16-bit element, 11 or 8 bits
// times 13) and of their sum (Knuth's, 6 operations) are added up with the low parts of c and s before
// the last rounding: 2^-37 of the larger product is what is lost before it.
template <typename T>
__device__ __forceinline__ float rotate_once(float x, float y, const Turn& t, float sign) {
  const float sh = sign * t.sh, sl = sign * t.sl;
  const float p = __fmul_rn(x, t.ch), q = __fmul_rn(y, sh);
  const float sum = __fadd_rn(p, q);
  const float b = __fsub_rn(sum, p);
  float low = __fadd_rn(__fsub_rn(p, __fsub_rn(sum, b)), __fsub_rn(q, b));
  if constexpr (sizeof(T) == 4)
    low = __fadd_rn(low, __fadd_rn(__fmaf_rn(x, t.ch, -p), __fmaf_rn(y, sh, -q)));
  low = __fmaf_rn(x, t.cl, __fmaf_rn(y, sl, low));
  return __fadd_rn(sum, low);
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
      turns[i] = make_turn<T>(position, a.freq[i], a.magnitude);
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
      return rotate_once<T>(own, to_f32(x[other]), turns[pair], second ? 1.f : -1.f);
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

// Codes 0 .. 2^bits - 1 (as floats) of 8 elements of one group: round-half-even(x / scale) + mid with
// the FP32 quotient. x times the scale's reciprocal is within 2e-6 of that quotient, so the rounding
// can only differ next to a border between two codes; there (and for anything not finite) the
// elements are divided.
template <int BITS>
__device__ __forceinline__ void quantize8(const float (&x)[8], float scale, float (&code)[8]) {
  constexpr float kMid = static_cast<float>(1 << (BITS - 1)), kRound = 12582912.f;  // 1.5 2^23
  const float inverse = __frcp_rn(scale);
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = __fmaf_rn(x[i], inverse, kMid);
    code[i] = __fsub_rn(__fadd_rn(y, kRound), kRound);
    far = max_nan(far, fabsf(y - code[i]));
  }
  if (!(far < 0.499998f)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int n = __float2int_rn(__fdiv_rn(x[i], scale));  // NaN: 0
      code[i] = static_cast<float>(max(-(1 << (BITS - 1)), min((1 << (BITS - 1)) - 1, n))) + kMid;
    }
  }
}

// Codes packed low bits first. Their weighted sum is a whole number below 2^16, exact in FP32.
template <int BITS>
__device__ __forceinline__ uint32_t pack8(const float (&code)[8]) {
  constexpr int kHalf = 16 / BITS;  // codes of 16 bits
  uint32_t part[8 / kHalf];
#pragma unroll
  for (int k = 0; k < 8 / kHalf; ++k) {
    float sum = code[k * kHalf + kHalf - 1];
#pragma unroll
    for (int i = kHalf - 2; i >= 0; --i)
      sum = __fmaf_rn(sum, static_cast<float>(1 << BITS), code[k * kHalf + i]);
    part[k] = __float_as_uint(sum + 8388608.f) & 0xFFFFu;
  }
  return BITS == 4 ? part[0] | part[8 / kHalf - 1] << 16 : part[0];
}

// Eight elements of a lane, as loaded.
template <typename T>
struct alignas(16) Eight {
  T e[8];
};

// A lane holds 8 consecutive elements of a row (head), a row is d / 8 lanes, a warp 32 / (d / 8) rows at
// a time; a task is kIters such steps over the heads of one token's keys or values, their loads all in
// flight at once. The cos and sin of the token's pairs are computed by the task's lanes and handed
// around through shared memory, then stay in registers over the heads; a rotation's other element comes
// from a lane of the same row (half layout) or is the lane's own (interleaved).
template <typename T, int BITS, bool INTERLEAVED, int kIters>
__global__ void __launch_bounds__(kThreads) append_rows_kernel(const AppendArgs a, int chunks) {
  extern __shared__ Turn turns[];  // [warps][pairs]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int lanes = a.d / 8, rows = 32 / lanes;  // lanes of a row, rows of a warp
  const int l = lane % lanes, row = lane / lanes;
  const int task = blockIdx.x * (kThreads / 32) + warp;
  const int per_token = 2 * chunks;
  const int token = task / per_token, kv = task % per_token / chunks, chunk = task % chunks;
  const int pairs = a.freq ? a.pairs : 0;
  pdl_wait();
  pdl_launch();
  if (token >= a.tokens) return;

  const RowTensor& in = kv ? a.value : a.key;
  const T* x = static_cast<const T*>(in.p) + token * in.token + l * 8;
  Eight<T> data[kIters];
  const int head0 = chunk * rows * kIters + row;
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    const int h = head0 + i * rows;
    if (row < rows && h < a.kvh) data[i] = *reinterpret_cast<const Eight<T>*>(x + h * in.head);
  }
  const long long slot = pool_row(a, index_at(a.slots, token));
  if (kv == 0 && chunk == 0 && lane == 0 && slot >= 0 && a.valid)
    atomicMax(a.valid + slot / a.bt, static_cast<int>(slot % a.bt) + 1);

  // the turns of this lane's elements; none for a value, or an element behind the rotated part
  constexpr int kTurns = INTERLEAVED ? 4 : 8;
  Turn turn[kTurns];
  float sign = 0.f;   // of the other element's sine: half layout
  int other = lane;   // the lane that holds it
  const bool turning = kv == 0 && pairs > 0;  // the same for the whole warp
  if (turning) {
    Turn* mine = turns + warp * pairs;
    const long long position = index_at(a.positions, token);
    for (int i = lane; i < pairs; i += 32) mine[i] = make_turn<T>(position, a.freq[i], a.magnitude);
    __syncwarp();
    const bool rotated = row < rows && l * 8 < 2 * pairs, second = l * 8 >= pairs;
    const int first = INTERLEAVED ? l * 4 : (second ? l * 8 - pairs : l * 8);
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      turn[i] = {1.f, 0.f, 0.f, 0.f};
      if (rotated) turn[i] = mine[first + i];
    }
    if (rotated && !INTERLEAVED) {
      other = second ? lane - pairs / 8 : lane + pairs / 8;
      sign = second ? 1.f : -1.f;
    }
  }
  const int group_lanes = a.group / 8, groups = a.d / a.group;
  const bool butterfly = (group_lanes & (group_lanes - 1)) == 0;
  constexpr float kMid = static_cast<float>(1 << (BITS - 1));
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    const int h = head0 + i * rows;
    if (h - row >= a.kvh) break;  // the same for the whole warp
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = to_f32(data[i].e[k]);
    if (turning) {
      float w[8];
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = rotate_once<T>(v[k], v[k ^ 1], turn[k / 2], k & 1 ? 1.f : -1.f);
      } else {
        Eight<T> there;
        const uint32_t* from = reinterpret_cast<const uint32_t*>(&data[i]);
        uint32_t* to = reinterpret_cast<uint32_t*>(&there);
#pragma unroll
        for (int k = 0; k < static_cast<int>(sizeof(Eight<T>) / 4); ++k)
          to[k] = __shfl_sync(0xffffffffu, from[k], other);
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = rotate_once<T>(v[k], to_f32(there.e[k]), turn[k], sign);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = w[k];
    }
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max_nan(top, fabsf(v[k]));
    if (butterfly) {
      for (int o = 1; o < group_lanes; o <<= 1)
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    } else {
      const int base = row * lanes + l / group_lanes * group_lanes;
      float all = top;
      for (int o = 0; o < group_lanes; ++o) all = max_nan(all, __shfl_sync(0xffffffffu, top, base + o));
      top = all;
    }
    const float scale = __fdiv_rn(max_nan(top, 1e-8f), kMid - 1.f);
    const __half held = __float2half_rn(scale);
    float code[8];
    quantize8<BITS>(v, scale, code);
    if (row >= rows || h >= a.kvh) continue;
    if (slot >= 0) {
      const long long at = slot * a.kvh + h;
      const uint32_t bytes = pack8<BITS>(code);
      uint8_t* codes = a.packed[kv] + at * (a.d * BITS / 8) + l * BITS;
      if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(codes) = bytes;
      else *reinterpret_cast<uint16_t*>(codes) = static_cast<uint16_t>(bytes);
      if (l % group_lanes == 0) a.scales[kv][at * groups + l / group_lanes] = held;
    }
    if (a.values[kv]) {
      const float unit = __half2float(held);
      Eight<__half> out;
#pragma unroll
      for (int k = 0; k < 8; ++k) out.e[k] = __float2half_rn(__fmul_rn(code[k] - kMid, unit));
      *reinterpret_cast<Eight<__half>*>(a.values[kv] + (static_cast<long long>(token) * a.kvh + h) * a.d +
                                        l * 8) = out;
    }
  }
}

template <typename T, int BITS, bool INTERLEAVED>
cudaError_t launch_rows(const AppendArgs& a, cudaStream_t s) {
  const int rows = 32 / (a.d / 8), warps = kThreads / 32;
  // Four steps a task keep 2 KB a warp in flight; with few tokens one step a task spreads the work
  // over more warps instead.
  const int long_chunks = (a.kvh + 4 * rows - 1) / (4 * rows), short_chunks = (a.kvh + rows - 1) / rows;
  const bool few = 2ll * a.tokens * long_chunks < 148 * 16;
  const int chunks = few ? short_chunks : long_chunks;
  const long long tasks = 2ll * a.tokens * chunks;
  if (tasks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  const size_t smem = a.freq ? static_cast<size_t>(warps) * a.pairs * sizeof(Turn) : 0;
  const auto kernel = few ? append_rows_kernel<T, BITS, INTERLEAVED, 1> : append_rows_kernel<T, BITS, INTERLEAVED, 4>;
  return launch_pdl(kernel, dim3(static_cast<unsigned>((tasks + warps - 1) / warps)), kThreads, smem, s,
                    a, chunks);
}

// Whether append_rows_kernel takes this call.
template <typename T>
bool by_rows(const AppendArgs& a) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.key.p) | reinterpret_cast<uintptr_t>(a.value.p) |
                       reinterpret_cast<uintptr_t>(a.values[0]) | reinterpret_cast<uintptr_t>(a.values[1]) |
                       reinterpret_cast<uintptr_t>(a.packed[0]) | reinterpret_cast<uintptr_t>(a.packed[1]);
  const long long strides = a.key.token | a.key.head | a.value.token | a.value.head;
  if (at % 16 || strides * static_cast<long long>(sizeof(T)) % 16 || a.d % 8 || a.group % 8) return false;
  return !a.freq || a.pairs % (a.interleaved ? 4 : 8) == 0;
}

template <typename T>
cudaError_t dispatch(const AppendArgs& a, cudaStream_t s) {
  if (by_rows<T>(a)) {
    if (a.bits == 4) return a.interleaved ? launch_rows<T, 4, true>(a, s) : launch_rows<T, 4, false>(a, s);
    return a.interleaved ? launch_rows<T, 2, true>(a, s) : launch_rows<T, 2, false>(a, s);
  }
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
