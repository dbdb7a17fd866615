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
// By its bytes bound by HBM: the inputs are read once, codes and scales (and, when asked for, the FP16
// values that the codes stand for) are written once. The arithmetic comes close to that time, so it works
// on two elements an instruction and divides by remainders. 8192 tokens x 8 heads x 128 BF16 to INT4:
// 15.2 us with the values written (floor 11.7); keys rotated 25.7 (FP32 keys 32.0, floor 16.8), bound by the
// latency of the rotation's chain at the 16 to 24 warps an SM that its registers leave (58 % of the issue
// slots are used; the four-step form of 16-bit types spills 12 bytes a thread at its 80 registers).
//
// append_rows_kernel: scale groups and pairs of whole 8 elements, rows on 16 bytes. append_kernel is
// the form for any other shape and alignment: a CTA takes one token, a warp one scale group after the
// other, a lane one byte of codes after the other.
#include "cache_ops.cuh"

namespace kvb {
namespace {

constexpr int kThreads = 256;

// (hi, lo) pairs of m cos t and m sin t.
struct alignas(16) Turn {
  float ch, cl, sh, sl;
};

// sin and cos of f turns, |f| <= 1/2, to 2^-44: the Taylor series on an eighth of a turn to either side
// of the nearest quarter (the first terms left out: x^15 / 15! and x^16 / 16! at pi / 4).
__device__ __forceinline__ void sin_cos(double f, double& s, double& c) {
  const double quarter = rint(4.0 * f);
  const double x = 6.283185307179586 * fma(-0.25, quarter, f), x2 = x * x;
  double a = 1.0 / 6227020800.0, b = -1.0 / 87178291200.0;
  a = fma(a, x2, -1.0 / 39916800.0);
  b = fma(b, x2, 1.0 / 479001600.0);
  a = fma(a, x2, 1.0 / 362880.0);
  b = fma(b, x2, -1.0 / 3628800.0);
  a = fma(a, x2, -1.0 / 5040.0);
  b = fma(b, x2, 1.0 / 40320.0);
  a = fma(a, x2, 1.0 / 120.0);
  b = fma(b, x2, -1.0 / 720.0);
  a = fma(a, x2, -1.0 / 6.0);
  b = fma(b, x2, 1.0 / 24.0);
  b = fma(b, x2, -0.5);
  a = fma(a * x2, x, x);
  b = fma(b, x2, 1.0);
  const int q = static_cast<int>(quarter) & 3;
  const double sin0 = q & 1 ? b : a, cos0 = q & 1 ? a : b;
  s = q & 2 ? -sin0 : sin0;
  c = (q + 1) & 2 ? -cos0 : cos0;
}

// A 16-bit element times ch must be exact in FP32 for rotate_once: ch then has 13 bits.
template <typename T>
__device__ __forceinline__ float high_part(double x) {
  const float f = static_cast<float>(x);
  return sizeof(T) == 2 ? __uint_as_float(__float_as_uint(f) & 0xFFFFF800u) : f;
}

template <typename T>
__device__ __forceinline__ Turn make_turn(long long position, double freq, float magnitude) {
  double s, c;
  sin_cos(turn_fraction(position, freq), s, c);
  c *= static_cast<double>(magnitude);
  s *= static_cast<double>(magnitude);
  Turn t;
  t.ch = high_part<T>(c);
  t.cl = static_cast<float>(c - static_cast<double>(t.ch));
  t.sh = high_part<T>(s);
  t.sl = static_cast<float>(s - static_cast<double>(t.sh));
  return t;
}

// x c + y s rounded once, for two elements: the rounding errors of the products (none for a 16-bit
// element, 11 or 8 bits times 13) and of their sum (Knuth's, 6 operations) are added up with the low
// parts of c and s before the last rounding: 2^-37 of the larger product is what is lost before it.
template <typename T>
__device__ __forceinline__ F2 rotate_once(F2 x, F2 y, F2 ch, F2 cl, F2 sh, F2 sl) {
  const F2 p = mul2(x, ch), q = mul2(y, sh);
  const F2 sum = add2(p, q);
  const F2 b = sub2(sum, p);
  F2 low = add2(sub2(p, sub2(sum, b)), sub2(q, b));
  if constexpr (sizeof(T) == 4)
    low = add2(low, add2(fma2(x, ch, mul2(p, f2(-1.f))), fma2(y, sh, mul2(q, f2(-1.f)))));
  low = fma2(x, cl, fma2(y, sl, low));
  return add2(sum, low);
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
      const Turn& t = turns[pair];
      const float sign = second ? 1.f : -1.f;
      return parts(rotate_once<T>(f2(own), f2(to_f32(x[other])), f2(t.ch), f2(t.cl), f2(sign * t.sh),
                                  f2(sign * t.sl))).x;
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

// 1 / x to half an ulp and a little: one Newton step from the hardware's approximation.
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return __fmaf_rn(__fmaf_rn(-x, r, 1.f), r, r);
}

// a / b rounded to nearest, given b's reciprocal: two steps of Markstein's (1990) from a * inverse, each
// adding the remainder (exact in an FMA) times the inverse; the first brings the quotient within an
// ulp, the second rounds it. The inverse must not be subnormal: b is below 2^126. Quotients here are 0 or
// far from FP32's limits.
__device__ __forceinline__ F2 quotient(F2 a, F2 b, F2 inverse) {
  const F2 minus = mul2(b, f2(-1.f));
  F2 q = mul2(a, inverse);
  q = fma2(fma2(minus, q, a), inverse, q);
  return fma2(fma2(minus, q, a), inverse, q);
}

// Quantizes 8 elements of one group: codes 0 .. 2^bits - 1 as floats. Adding 1.5 2^23 + mid rounds the
// quotient half to even and adds the (even) midpoint. An INT4 scale is below 2^128 / 7; an INT2 one may be
// any finite number, so its quotients are taken by a quarter of it, and divided by 4 as they are rounded.
template <int BITS>
__device__ __forceinline__ void quantize8(const F2 (&x)[4], float scale, F2 (&code)[4]) {
  constexpr float kPart = BITS == 2 ? 0.25f : 1.f;
  const F2 round = f2(12582912.f + (1 << (BITS - 1)));
  const F2 b = f2(scale * kPart), inverse = f2(reciprocal(scale * kPart));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const F2 q = quotient(x[i], b, inverse);
    code[i] = add2(BITS == 2 ? fma2(q, f2(kPart), round) : add2(q, round), f2(-12582912.f));
  }
}

// max|x| / (2^(bits-1) - 1), at least 1e-8 over that.
template <int BITS>
__device__ __forceinline__ float scale_of(float top) {
  top = max_nan(top, 1e-8f);
  if constexpr (BITS == 2) return top;
  const float scale = parts(quotient(f2(top), f2(7.f), f2(1.f / 7.f))).x;
  return top < INFINITY ? scale : top;  // an infinity or a NaN shows in the scale
}

// Codes packed low bits first. Weighted sums of codes are whole numbers below 2^16, exact in FP32.
template <int BITS>
__device__ __forceinline__ uint32_t pack8(const F2 (&code)[4]) {
  // even codes in one half, odd ones in the other
  constexpr float kStep = static_cast<float>(1 << (2 * BITS)), kOdd = static_cast<float>(1 << BITS);
  const auto word = [&](F2 sum) {
    const float2 two = parts(sum);
    return __float_as_uint(__fmaf_rn(two.y, kOdd, two.x) + 8388608.f) & 0xFFFFu;
  };
  const F2 low = fma2(code[1], f2(kStep), code[0]), high = fma2(code[3], f2(kStep), code[2]);
  if constexpr (BITS == 4) return word(low) | word(high) << 16;
  return word(fma2(high, f2(kStep * kStep), low));
}

// Eight elements of a lane, as loaded.
template <typename T>
struct alignas(16) Eight {
  static constexpr int kWords = 2 * sizeof(T);
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; i += 4)
      *reinterpret_cast<uint4*>(w + i) = reinterpret_cast<const uint4*>(p)[i / 4];
  }
};

// A lane holds 8 consecutive elements of a row (head), a row is d / 8 lanes, a warp takes `heads` rows at a
// time; a task is kIters such steps over the heads of one token's keys or values, their loads all in flight
// at once. Where one step takes all heads and leaves half of a warp's lanes or more without work, a task is
// that step of `per_warp` tokens (8.4 M elements, one head of 64: 59 us, with one token a warp 244). The cos
// and sin of a token's pairs are computed by the task's lanes and handed around through shared memory, then
// stay in registers over the heads; a rotation's other element comes from a lane of the same row (half
// layout) or is the lane's own (interleaved). kGroupLanes: the lanes of a scale group, 0: any number.
// TURNS: whether a task's keys may be rotated; the kernel without it needs half the registers.
constexpr int resident(int iters, int bytes, bool turns) {
  return turns ? (bytes == 2 ? 3 : 2) : (bytes == 2 ? 4 : 3);
}

template <typename T, int BITS, bool INTERLEAVED, int kIters, int kGroupLanes, bool TURNS>
__global__ void __launch_bounds__(kThreads, resident(kIters, sizeof(T), TURNS))
    append_rows_kernel(const AppendArgs a, unsigned per_lane, int heads, int per_warp) {
  extern __shared__ Turn turns[];  // [warps][per_warp][pairs]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int lanes = a.d >> 3;                                   // of a row
  const int row = lane * per_lane >> 16;  // of the warp
  const int l = lane - row * lanes;
  const int step = kIters == 1 ? heads : 32u * per_lane >> 16;  // several steps use all of a warp's rows
  const int tokens = kIters == 1 ? per_warp : 1;  // of the warp
  const int nth = kIters == 1 ? row / step : 0, step_row = row - nth * step;
  const int kv = blockIdx.y & 1, chunk = blockIdx.y >> 1;
  const int token0 = (blockIdx.x * (kThreads / 32) + warp) * tokens, token = token0 + nth;
  const int pairs = a.freq ? a.pairs : 0;
  pdl_wait();
  pdl_launch();
  if (token0 >= a.tokens) return;
  const bool live = kIters == 1 ? nth < tokens && token < a.tokens : row < step;  // lanes with a row

  const RowTensor& in = kv ? a.value : a.key;
  const T* x = static_cast<const T*>(in.p) + token * in.token + l * 8;
  Eight<T> data[kIters];
  const int head0 = chunk * step * kIters + step_row;
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    const int h = head0 + i * step;
    if (live && h < a.kvh) data[i].load(x + h * in.head);
    else data[i] = {};
  }
  const long long slot = live ? pool_row(a, index_at(a.slots, token)) : -1;
  if (kv == 0 && chunk == 0 && step_row == 0 && l == 0 && slot >= 0 && a.valid) {
    // below 2^32 rows (nearly always) the division is the short one
    const long long block = slot >> 32 ? slot / a.bt : static_cast<unsigned>(slot) / static_cast<unsigned>(a.bt);
    atomicMax(a.valid + block, static_cast<int>(slot - block * a.bt) + 1);
  }

  // the turns of this lane's elements, in pairs of elements, signs included; no turn for an element
  // behind the rotated part
  F2 ch[4], cl[4], sh[4], sl[4];
  int other = lane;  // the lane that holds the pairs' other elements: half layout
  const bool turning = TURNS && kv == 0 && pairs > 0;  // the same for the whole warp
  if (turning) {
    Turn* mine = turns + warp * tokens * pairs;
    // pair i at (i % kRun) * (pairs / kRun) + i / kRun: lanes read consecutive entries
    constexpr int kRun = INTERLEAVED ? 4 : 8;
    const int runs = pairs / kRun;
    for (int t = 0; t == 0 || (kIters == 1 && t < tokens && token0 + t < a.tokens); ++t) {
      const long long position = index_at(a.positions, token0 + t);
      for (int i = lane; i < pairs; i += 32)
        mine[t * pairs + i % kRun * runs + i / kRun] = make_turn<T>(position, a.freq[i], a.magnitude);
    }
    __syncwarp();
    const bool rotated = live && l * 8 < 2 * pairs, second = l * 8 >= pairs;
    const Turn* own = mine + nth * pairs + (INTERLEAVED || !second ? l : l - pairs / 8);
    const float sign = second ? 1.f : -1.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ch[i] = f2(1.f), cl[i] = sh[i] = sl[i] = f2(0.f);
      if (!rotated) continue;
      if constexpr (INTERLEAVED) {
        const Turn t = own[i * runs];
        ch[i] = f2(t.ch), cl[i] = f2(t.cl), sh[i] = f2(-t.sh, t.sh), sl[i] = f2(-t.sl, t.sl);
      } else {
        const Turn t = own[2 * i * runs], u = own[(2 * i + 1) * runs];
        ch[i] = f2(t.ch, u.ch), cl[i] = f2(t.cl, u.cl);
        sh[i] = f2(sign * t.sh, sign * u.sh), sl[i] = f2(sign * t.sl, sign * u.sl);
      }
    }
    if (rotated && !INTERLEAVED) other = second ? lane - pairs / 8 : lane + pairs / 8;
  }
  const int group_lanes = kGroupLanes ? kGroupLanes : a.group / 8, groups = a.d / a.group;
  constexpr float kMid = static_cast<float>(1 << (BITS - 1));
  // this lane's outputs of its first head; those of the next are rows heads on
  const long long at = slot * a.kvh + head0;
  uint8_t* codes = a.packed[kv] + at * (lanes * BITS) + l * BITS;
  __half* scales = a.scales[kv] + at * groups + l / group_lanes;
  const bool leads = l == l / group_lanes * group_lanes;
  __half* values = a.values[kv];
  if (values) values += ((static_cast<long long>(token) * a.kvh + head0) * lanes + l) * 8;
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    // no early end: the iterations' chains of dependent operations overlap
    const bool mine = live && head0 + i * step < a.kvh;
    F2 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = unpack_pair<T>(data[i].w, k);
    if (turning) {
      Eight<T> there;
      if constexpr (!INTERLEAVED) {
#pragma unroll
        for (int k = 0; k < Eight<T>::kWords; ++k)
          there.w[k] = __shfl_sync(0xffffffffu, data[i].w[k], other);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        F2 w;
        if constexpr (INTERLEAVED) {
          const float2 two = parts(v[k]);
          w = f2(two.y, two.x);
        } else {
          w = unpack_pair<T>(there.w, k);
        }
        v[k] = rotate_once<T>(v[k], w, ch[k], cl[k], sh[k], sl[k]);
      }
    }
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 two = parts(v[k]);
      top = max_nan(top, max_nan(fabsf(two.x), fabsf(two.y)));
    }
    if constexpr (kGroupLanes > 0) {
#pragma unroll
      for (int o = 1; o < kGroupLanes; o <<= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    } else {
      const int base = row * lanes + l / group_lanes * group_lanes;
      const float own = top;
      for (int o = 0; o < group_lanes; ++o) top = max_nan(top, __shfl_sync(0xffffffffu, own, base + o));
    }
    const float scale = scale_of<BITS>(top);
    const __half held = __float2half_rn(scale);
    F2 code[4];
    quantize8<BITS>(v, scale, code);
    const uint32_t bytes = pack8<BITS>(code);
    uint8_t* to = codes + i * (step * lanes * BITS);
    if (mine && slot >= 0) {
      if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(to) = bytes;
      else *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(bytes);
    }
    if (mine && slot >= 0 && leads) scales[i * (step * groups)] = held;
    if (mine && values) {
      const F2 unit = f2(__half2float(held));
      uint32_t out[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) pack_pair<__half>(mul2(add2(code[k], f2(-kMid)), unit), out, k);
      *reinterpret_cast<uint4*>(values + i * (step * lanes * 8)) = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
}

template <typename T, int BITS, bool INTERLEAVED, int kIters>
cudaError_t launch_iters(const AppendArgs& a, int step, int per_warp, cudaStream_t s) {
  const int warps = kThreads / 32, chunks = (a.kvh + kIters * step - 1) / (kIters * step);
  // lane / lanes as a product: 2^16 / lanes rounded up is exact for 32 lanes
  const unsigned per_lane = (65536u + a.d / 8 - 1) / (a.d / 8);
  const dim3 grid((a.tokens + warps * per_warp - 1) / (warps * per_warp), 2 * chunks);
  const bool g32 = a.group == 32;
  // Keys that do not turn take the kernel that needs half the registers (8192 tokens: 14.8 us, by the kernel
  // that can turn 18.5). Where they do turn, values in a launch of their own are slower (25.9 us for 24.6;
  // 2048 tokens 13.1 for 8.8).
  if (!a.freq)
    return launch_pdl(g32 ? append_rows_kernel<T, BITS, false, kIters, 4, false>
                          : append_rows_kernel<T, BITS, false, kIters, 0, false>,
                      grid, kThreads, 0, s, a, per_lane, step, per_warp);
  const size_t smem = static_cast<size_t>(warps) * per_warp * a.pairs * sizeof(Turn);
  return launch_pdl(g32 ? append_rows_kernel<T, BITS, INTERLEAVED, kIters, 4, true>
                        : append_rows_kernel<T, BITS, INTERLEAVED, kIters, 0, true>,
                    grid, kThreads, smem, s, a, per_lane, step, per_warp);
}

template <typename T, int BITS, bool INTERLEAVED>
cudaError_t launch_rows(const AppendArgs& a, cudaStream_t s) {
  // Heads a warp takes at a time, and steps to take them all. Up to four steps a task keep 2 KB a warp in
  // flight, no more than there are heads for (4 heads of 128: two steps 30.2 us, four 39.7). One step a task
  // spreads the work of few tokens over more warps: up to 32 an SM (8 heads of 128, 128 tokens: one step
  // 3.4 us, four 4.7; 450: 4.7 both; 1100: 7.8 and 6.6. One head of 64, 600 tokens: 3.1 us, four tokens a
  // warp 3.9; 2400: 4.9 and 4.7).
  const int rows = 32 / (a.d / 8), step = rows < a.kvh ? rows : a.kvh, steps = (a.kvh + step - 1) / step;
  const bool few = 2ll * a.tokens * steps < 148 * 32;
  if (few) return launch_iters<T, BITS, INTERLEAVED, 1>(a, step, 1, s);
  if (steps == 1) return launch_iters<T, BITS, INTERLEAVED, 1>(a, step, rows / step, s);
  if (steps == 2) return launch_iters<T, BITS, INTERLEAVED, 2>(a, step, 1, s);
  return launch_iters<T, BITS, INTERLEAVED, 4>(a, step, 1, s);
}

// Whether append_rows_kernel takes this call.
template <typename T>
bool by_rows(const AppendArgs& a) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.key.p) | reinterpret_cast<uintptr_t>(a.value.p) |
                       reinterpret_cast<uintptr_t>(a.values[0]) | reinterpret_cast<uintptr_t>(a.values[1]) |
                       reinterpret_cast<uintptr_t>(a.packed[0]) | reinterpret_cast<uintptr_t>(a.packed[1]);
  const long long strides = a.key.token | a.key.head | a.value.token | a.value.head;
  if (at % 16 || strides * static_cast<long long>(sizeof(T)) % 16 || a.d % 8 || a.group % 8) return false;
  if (a.kvh > 16384) return false;  // the grid's second dimension
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
