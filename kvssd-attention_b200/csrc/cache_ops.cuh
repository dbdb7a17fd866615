// Cache-maintenance operators around the decode attention: rotary positions (rotary.cu), the
// quantizing cache write (append.cu), attention weights over the packed keys (weights.cu) and
// eviction by them (evict.cu). Launch arguments, the functions cache_api.cu calls, and the device
// helpers the kernels share.
//
// Every kernel is launched with programmatic stream serialization: its first instruction that
// touches global memory comes after pdl_wait().
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace kvb {

// A [tokens, heads, head_dim] tensor: strides in elements, the last dimension contiguous.
struct RowTensor {
  const void* p;
  long long token, head;
};

// int32 or int64 indices.
struct Indices {
  const void* p;
  int wide;  // 1: int64
};

struct RotaryArgs {
  RowTensor x;
  void* out;
  long long out_token, out_head;
  int dtype;
  int tokens, heads, d;
  Indices positions;
  const double* freq;  // radians a position, [pairs]
  int pairs, interleaved;
  float magnitude;
};

struct AppendArgs {
  RowTensor key, value;
  int dtype;
  int tokens;
  Indices slots, positions;
  const double* freq;  // nullptr: keys are stored as they are
  int pairs, interleaved;
  float magnitude;
  uint8_t* packed[2];  // K, V
  __half* scales[2];
  __half* values[2];   // nullptr, or FP16 [tokens, kvh, d]
  int32_t* valid;      // nullptr, or [n_pool]
  int n_pool, bt, kvh, d, bits, group;
  unsigned* status;    // nullptr, or the sticky status word
};

struct WeightsArgs {
  const void* query;
  int dtype;
  int queries, qh;
  const uint8_t* kp;
  const __half* ks;
  const int32_t* valid;
  const int32_t* table;    // nullptr: slots 0 .. n_sel - 1
  const int32_t* visible;  // nullptr: every query sees every place
  int n_pool, n_sel, bt, kvh, d, bits, group;
  float sm_scale;
  const float* lse_in;     // nullptr: computed
  float* lse;              // [queries, qh], written when computed
  const float* previous;   // nullptr, or [kvh, n_sel * bt] with this row stride
  long long previous_stride;
  float* out;
  long long out_stride;
  float* scratch;          // parts of the log-sum-exps when computed
  long long parts_room;    // as many a query row as it holds
  unsigned* status;
};

struct EvictArgs {
  const float* weights;
  long long weights_stride;
  const int32_t* positions;
  long long positions_stride;
  int n, keep, columns;    // columns of the outputs
  int sink;                // positions below are kept
  long long recent_from;   // positions from here on are kept
  int shared;
  float* new_weights;      // [kvh, columns]
  int32_t* new_positions;  // [kvh, columns]
  int32_t* holes;          // scratch [lists, keep]
  int32_t* movers;         // scratch [lists, n - keep]
  int32_t* counts;         // scratch [lists]
  unsigned* keys;          // scratch [lists, n] of the longest caches
  uint8_t* packed[2];
  __half* scales[2];
  int32_t* valid;
  const int32_t* table;
  int n_pool, n_sel, bt, kvh;
  int packed_dim, groups;  // bytes of codes and scales of one (token, head)
  unsigned* status;
};

// Sets the calling thread's last error and returns `status` (api.cu).
int report(int status, const char* message);

cudaError_t launch_rotary(const RotaryArgs& a, cudaStream_t s);
cudaError_t launch_append(const AppendArgs& a, cudaStream_t s);
size_t weights_scratch_bytes(int queries, int qh, int kvh, int n_sel, int bt, int d, int group);
cudaError_t launch_weights(const WeightsArgs& a, cudaStream_t s);
size_t evict_scratch_ints(int n, int lists);
cudaError_t launch_evict(const EvictArgs& a, cudaStream_t s);

// Launch with programmatic stream serialization (see above).
template <typename... Params, typename... Given>
cudaError_t launch_pdl(void (*kernel)(Params...), dim3 grid, int threads, size_t smem,
                       cudaStream_t s, Given... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

// n / d for 0 <= n < 2^31 as a product and a shift (Granlund and Montgomery, 1994).
struct Divisor {
  unsigned factor, shift;
};
inline Divisor divisor(unsigned d) {
  unsigned shift = 0;
  while ((1ull << shift) < d) ++shift;
  return {static_cast<unsigned>((((1ull << shift) - d) << 32) / d + 1), shift};
}
__device__ __forceinline__ int divide(int n, Divisor d) {
  return static_cast<int>((__umulhi(static_cast<unsigned>(n), d.factor) + static_cast<unsigned>(n)) >> d.shift);
}

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ long long index_at(const Indices& ix, long long i) {
  return ix.wide ? static_cast<const long long*>(ix.p)[i] : static_cast<const int32_t*>(ix.p)[i];
}

// Element types of the rotary and append operators.
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// The angle of `position` at `freq` radians a position, as a fraction of a turn in [-1/2, 1/2].
// The angle is the FP64 product; its division by 2 pi keeps the product's low part (1 / (2 pi) as
// a pair of doubles), so a far position loses nothing against reducing the FP64 angle exactly.
__device__ __forceinline__ double turn_fraction(long long position, double freq) {
  constexpr double kInv2PiHi = 0.15915494309189535;        // fl64(1 / (2 pi))
  constexpr double kInv2PiLo = -9.839338337591243e-18;     // 1 / (2 pi) - kInv2PiHi
  const double angle = static_cast<double>(position) * freq;
  const double hi = angle * kInv2PiHi;
  const double lo = fma(angle, kInv2PiHi, -hi) + angle * kInv2PiLo;
  return (hi - rint(hi)) + lo;
}

// Two FP32 numbers in one register pair: one instruction rounds both (PTX add/mul/fma.rn.f32x2).
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ F2 f2(float a) { return f2(a, a); }
__device__ __forceinline__ float2 parts(F2 x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// a - b: the product with -1 is exact.
__device__ __forceinline__ F2 sub2(F2 a, F2 b) { return fma2(b, f2(-1.f), a); }

// Vectors of N elements as 32-bit words: pairs of 16-bit elements are taken apart and put together a word
// at a time (arrays of 16-bit elements cost a register and several instructions each).
template <typename T>
__device__ __forceinline__ F2 unpack_pair(const uint32_t* w, int i);
template <>
__device__ __forceinline__ F2 unpack_pair<float>(const uint32_t* w, int i) {
  return f2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
}
template <>
__device__ __forceinline__ F2 unpack_pair<__half>(const uint32_t* w, int i) {
  const float2 two = __half22float2(u32_as_h2(w[i]));
  return f2(two.x, two.y);
}
template <>
__device__ __forceinline__ F2 unpack_pair<__nv_bfloat16>(const uint32_t* w, int i) {
  return f2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
}
template <typename T>
__device__ __forceinline__ void pack_pair(F2 x, uint32_t* w, int i);
template <>
__device__ __forceinline__ void pack_pair<float>(F2 x, uint32_t* w, int i) {
  const float2 two = parts(x);
  w[2 * i] = __float_as_uint(two.x);
  w[2 * i + 1] = __float_as_uint(two.y);
}
template <>
__device__ __forceinline__ void pack_pair<__half>(F2 x, uint32_t* w, int i) {
  const float2 two = parts(x);
  w[i] = h2_as_u32(__floats2half2_rn(two.x, two.y));
}
template <>
__device__ __forceinline__ void pack_pair<__nv_bfloat16>(F2 x, uint32_t* w, int i) {
  const float2 two = parts(x);
  const __nv_bfloat162 b = __floats2bfloat162_rn(two.x, two.y);
  memcpy(w + i, &b, 4);
}

}  // namespace kvb
