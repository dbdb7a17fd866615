// Tensor-core kernels of the attention weights (weights.cu), for head_dim 64, 96, 128 and 256 and
// scale groups of whole 16 dims.
//
// Math. A warp takes tiles of 16 (or 32) places of one KV head: S = K Q^T with mma.sync m16n8k16,
// 16 places by 8 query rows. The codes enter as exact centred FP16 integers and the queries as FP16, each
// row scaled by a power of two to the top of FP16's range: FP16 and BF16 ones as they are but for a rounding
// at 2^-39 of the row's largest, FP32 and FP64 ones as a high and a low part, 22 bits. Products are exact
// then and sums FP32; the FP16 key scales are constant over a unit of 32 (or 16) dims and multiply the
// unit's partial sums in FP32. Exponentials are ex2.approx, log-sum-exps pass through base 2 in FP32.
// More than 32 rows go to tcgen05 (weights_umma.cuh): its tiles are 128 rows wide however few are used.
// 65536 tokens x 8 heads x 128 INT4, log-sum-exps computed: 16 rows 52 us and 32 rows 69 us here, 64 rows
// 103 us and 128 rows 118 us there.
//
// Unit layout. A lane (r, c) of the A fragment holds the codes of row r (and r + 8) that lie c-th of
// four in the unit: 8 codes of a 32-dim unit, 4 of a 16-dim unit, unpacked two at a time into pairs
// p = (dim i, dim i + half): dims 8c + p and 8c + p + 4 (or 4c + p, 4c + p + 2). The B fragments hold
// the queries in the same order.
#pragma once

#include "cache_ops.cuh"

namespace kvb {
namespace weights_tc {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -1e30f;  // running max of a row that has seen nothing

enum Mode {
  kWindow,  // weights
  kLse      // parts (m, l) of up to kLseTiles tiles of query rows
};
constexpr int kLseTiles = 4;

struct Job {
  WeightsArgs a;
  int total_tiles;      // of 16 * MT places, of the whole selection
  int tiles_per_block;
  int tiles_per_cta;
  int heads_per_cta;    // of the step kernel
  int rows;             // query rows a KV head: queries * gqa
  int row0, row_tiles;  // the rows of this launch: row0 .. row0 + 8 row_tiles
  int parts;            // parts per row in scratch (0: lse given)
  int add;              // add to what out holds (later launches over more rows)
};

template <int BITS, int D, int UNIT>
struct Shape {
  static constexpr int kUnits = D / UNIT;
  static constexpr int kPairs = UNIT / 8;            // pairs a lane, row and unit
  static constexpr int kRowBytes = D * BITS / 8;
  static constexpr int kChunk = kRowBytes % 16 ? 8 : 16;  // bytes a copy
  static constexpr int kChunks = kRowBytes / kChunk;
  // Chunk q of row r is stored at chunk q ^ swizzle(r): the 8 rows of a fragment's load fall on
  // distinct banks (rows of 48 and 24 bytes do so by themselves).
  static constexpr bool kSwizzled = kRowBytes == 32 || kRowBytes == 64 || kRowBytes == 128;
  __device__ static __forceinline__ int swizzle(int r) {
    if constexpr (kSwizzled) return (r / (128 / kRowBytes)) & (kChunks - 1);
    return 0;
  }
};

// Centred codes of one lane, row and unit as exact FP16 pairs.
template <int BITS, int UNIT>
__device__ __forceinline__ void unpack(uint32_t x, uint32_t (&p)[UNIT / 8]) {
  if constexpr (BITS == 4 && UNIT == 32) {
    __half2 o[4];
    LanePairs<4>::centred(x, o);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = h2_as_u32(o[i]);
  } else if constexpr (BITS == 4) {  // 16 bits: bytes apart, so a lane of the word holds 2 codes
    const uint32_t y = __byte_perm(x, 0, 0x4140);
    p[0] = h2_as_u32(__hsub2(u32_as_h2(or_magic<0x000F000Fu>(y)), h2_const(0x64086408u)));
    p[1] = h2_as_u32(__hfma2(u32_as_h2(or_magic<0x00F000F0u>(y)), h2_const(0x2C002C00u),
                             h2_const(0xD480D480u)));
  } else {
    const uint32_t y = UNIT == 32 ? __byte_perm(x, 0, 0x4140) : (x | (x << 12));
    p[0] = h2_as_u32(__hsub2(u32_as_h2(or_magic<0x00030003u>(y)), h2_const(0x64026402u)));
    p[1] = h2_as_u32(__hfma2(u32_as_h2(or_magic<0x000C000Cu>(y)), h2_const(0x34003400u),
                             h2_const(0xDC08DC08u)));
    if constexpr (UNIT == 32) {
      p[2] = h2_as_u32(__hfma2(u32_as_h2(or_magic<0x00300030u>(y)), h2_const(0x2C002C00u),
                               h2_const(0xD420D420u)));
      p[3] = h2_as_u32(__hfma2(u32_as_h2(or_magic<0x00C000C0u>(y)), h2_const(0x24002400u),
                               h2_const(0xCC80CC80u)));
    }
  }
}

// The FP16 scales of one row, two to a word: of its groups as loaded, or one per unit.
template <int UNITS>
struct RowScales {
  uint32_t w[(UNITS + 1) / 2];
};

// Loads the `groups` scales of a row (the same number for all threads: the branches are uniform).
// Nothing here waits for the loads: they are spread over the units when the tile is used.
template <int UNITS>
__device__ __forceinline__ void load_scales(const __half* p, int groups, RowScales<UNITS>& s) {
  constexpr int W = (UNITS + 1) / 2;
  if (groups % 8 == 0) {
#pragma unroll
    for (int i = 0; i < W / 4; ++i)
      if (8 * i < groups) {
        const uint4 v = *reinterpret_cast<const uint4*>(p + 8 * i);
        s.w[4 * i] = v.x, s.w[4 * i + 1] = v.y, s.w[4 * i + 2] = v.z, s.w[4 * i + 3] = v.w;
      }
  } else if (groups == 4) {
    if constexpr (W >= 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      s.w[0] = v.x, s.w[1] = v.y;
    }
  } else if (groups % 2 == 0) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (2 * i < groups) s.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
  } else if (groups == 1) {
    s.w[0] = *reinterpret_cast<const unsigned short*>(p);
  } else {  // 3
    const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
    if constexpr (W >= 2) {
      s.w[0] = u[0] | static_cast<uint32_t>(u[1]) << 16;
      s.w[1] = u[2];
    }
  }
}

// Unit u takes the scale of group u / PER.
template <int UNITS, int PER>
__device__ __forceinline__ RowScales<UNITS> spread_by(const RowScales<UNITS>& g) {
  constexpr int W = (UNITS + 1) / 2;
  RowScales<UNITS> s;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const int u0 = 2 * i / PER, u1 = (2 * i + 1) / PER;
    const uint32_t lo = u0 & 1 ? g.w[u0 / 2] >> 16 : g.w[u0 / 2] & 0xFFFFu;
    s.w[i] = u1 / 2 < W ? lo | (u1 & 1 ? g.w[u1 / 2] & 0xFFFF0000u : g.w[u1 / 2] << 16) : lo;
  }
  return s;
}

template <int UNITS>
__device__ __forceinline__ RowScales<UNITS> spread(const RowScales<UNITS>& g, int groups) {
  const int per = UNITS / groups;
  if (per == 1) return g;
  if (per == 2) return spread_by<UNITS, 2>(g);
  if (per == 3) return spread_by<UNITS, 3>(g);
  if (per == 4) return spread_by<UNITS, 4>(g);
  if (per == 8) return spread_by<UNITS, 8>(g);
  return spread_by<UNITS, 16>(g);  // one group: 6 or 16 units
}

// Whether query t of query head `head` adds to any place. One that sees nothing, or whose given
// log-sum-exp says so, may hold anything (padding): it enters the products as zeros.
__device__ __forceinline__ bool adds(const WeightsArgs& a, int t, int head) {
  return !(a.visible && a.visible[t] <= 0) &&
         !(a.lse_in && a.lse_in[static_cast<long long>(t) * a.qh + head] == -INFINITY);
}

// The B fragments of 8 query rows (lane: row lane / 4) and the factor that turns their sums into
// scores in the log2 domain: sm_scale log2(e) / 2^e, with 2^e the row's scale.
template <int D, int UNIT, bool LO>
struct QueryTile {
  static constexpr int kUnits = D / UNIT, kPairs = UNIT / 8;
  uint32_t b[(LO ? 2 : 1) * kUnits][kPairs];  // high parts, then low parts
  float factor;

  __device__ __forceinline__ void load(const Job& j, int h, int tile, int lane) {
    const WeightsArgs& a = j.a;
    const int gqa = a.qh / a.kvh, row = j.row0 + 8 * tile + (lane >> 2), c = lane & 3;
    constexpr int kOwn = UNIT / 4;  // dims a lane holds of a unit
    float q[kUnits][kOwn];
    float top = 0.f;
    if (row < j.rows) {
      const long long at = (static_cast<long long>(row / gqa) * a.qh + h * gqa + row % gqa) * D;
      const bool live = adds(a, row / gqa, h * gqa + row % gqa);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if constexpr (kOwn == 8) {
          load_query8(a.query, a.dtype, at + u * UNIT + c * kOwn, q[u]);
        } else {
#pragma unroll
          for (int i = 0; i < kOwn; ++i) q[u][i] = load_query(a.query, a.dtype, at + u * UNIT + c * kOwn + i);
        }
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          if (!live) q[u][i] = 0.f;
          top = fmaxf(top, fabsf(q[u][i]));
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
#pragma unroll
        for (int i = 0; i < kOwn; ++i) q[u][i] = 0.f;
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^e brings the row's largest element into [2^14, 2^15); e in two steps, since 2^e alone can
    // leave FP32's range
    int e = 0;
    if (top > 0.f && top < INFINITY) e = 14 - ilogbf(top);
    const auto power = [](int i) { return __int_as_float((i + 127) << 23); };
    const int e1 = e / 2, e2 = e - e1;
    const float s1 = power(e1), s2 = power(e2);
    factor = a.sm_scale * kLog2e * power(-e1) * power(-e2);
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
#pragma unroll
      for (int p = 0; p < kPairs; ++p) {
        const float x = q[u][p] * s1 * s2, y = q[u][p + kPairs] * s1 * s2;
        const __half hx = __float2half_rn(x), hy = __float2half_rn(y);
        b[u][p] = h2_as_u32(__halves2half2(hx, hy));
        if constexpr (LO)
          b[kUnits + u][p] = h2_as_u32(__floats2half2_rn(x - __half2float(hx), y - __half2float(hy)));
      }
  }
};

// A log-sum-exp in the log2 domain, as the weights subtract it: +inf where the row adds nothing.
__device__ __forceinline__ float as_log2(float lse) {
  return lse == -INFINITY ? INFINITY : lse * kLog2e;
}

// All lanes: (m, l) of query row `row` of head h from its parts, as its log-sum-exp in the log2
// domain (m in log2 units); -inf for a row that has seen nothing.
__device__ __forceinline__ float combine_parts(const Job& j, int h, int row, int lane) {
  const float2* part = reinterpret_cast<const float2*>(j.a.scratch) +
                       (static_cast<long long>(h) * j.rows + row) * j.parts;
  float m = kLowest, l = 0.f;
  for (int p = lane; p < j.parts; p += 32) {
    const float2 v = part[p];
    const float top = fmaxf(m, v.x);
    l = l * fast_exp2(m - top) + v.y * fast_exp2(v.x - top);
    m = top;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
    const float top = fmaxf(m, m2);
    l = l * fast_exp2(m - top) + l2 * fast_exp2(m2 - top);
    m = top;
  }
  return l == 0.f ? -INFINITY : m + log2f(l);
}

// One lane's fragment of one unit from shared memory, in one access.
__device__ __forceinline__ void load_fragment(const uint32_t (&from)[4], uint32_t (&b)[4]) {
  const uint4 v = *reinterpret_cast<const uint4*>(from);
  b[0] = v.x, b[1] = v.y, b[2] = v.z, b[3] = v.w;
}
__device__ __forceinline__ void load_fragment(const uint32_t (&from)[2], uint32_t (&b)[2]) {
  const uint2 v = *reinterpret_cast<const uint2*>(from);
  b[0] = v.x, b[1] = v.y;
}

// mma_16816 with the sum's start in registers of its own, (c0, c1) for both rows.
__device__ __forceinline__ void mma_16816_from(float (&d)[4], float c0, float c1, uint32_t a0,
                                               uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}

// What the weights kernels keep of a query row.
struct alignas(8) RowInfo {
  float factor, lse2;
};

// CTAs along the places for `total` tiles of kvh heads, `heads` of them a CTA of `warps` warps: as many
// as are resident at once, each with a contiguous run of tiles.
inline int grid_x(int total, int kvh, int heads, int warps, int ctas) {
  const int subs = warps / heads, ys = kvh / heads;
  const int most = (total + subs - 1) / subs, want = 148 * ctas / ys;
  return want < 1 ? 1 : (want < most ? want : most);
}

}  // namespace weights_tc

// Launchers, one translation unit per head_dim.
cudaError_t launch_weights_tc_64(const WeightsArgs& a, cudaStream_t s);
cudaError_t launch_weights_tc_96(const WeightsArgs& a, cudaStream_t s);
cudaError_t launch_weights_tc_128(const WeightsArgs& a, cudaStream_t s);
cudaError_t launch_weights_tc_256(const WeightsArgs& a, cudaStream_t s);
}  // namespace kvb
