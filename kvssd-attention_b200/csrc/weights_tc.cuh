// Tensor-core kernels of the attention weights (weights.cu), for head_dim 64, 96, 128 and 256 and
// scale groups of whole 16 dims.
//
// Math. A warp takes tiles of 16 (or 32) places of one KV head: S = K Q^T with mma.sync m16n8k16,
// 16 places by 8 query rows. The codes enter as exact centred FP16 integers and the queries as FP16
// (FP32 and FP64 ones as a high and a low part), each row scaled by a power of two to the top of
// FP16's range, so that every product is exact and the FP32 sums are the only rounding; the FP16 key
// scales are constant over a unit of 32 (or 16) dims and multiply the unit's partial sums in FP32.
// tcgen05 would need the dequantized FP16 keys in shared memory and a scale per row and unit between
// its MMAs (none of its block scalings is FP16 per 16 or 32 elements), and at one decode step's 4 to
// 8 query rows a unit the tensor work is a tenth of the copies' time.
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
  kStep,    // weights, one tile of 8 query rows held in registers
  kWindow,  // weights, any number of query rows, their fragments in shared memory
  kLse      // parts (m, l) of up to kLseTiles tiles of query rows
};
constexpr int kLseTiles = 4;

struct Job {
  WeightsArgs a;
  int total_tiles;      // of 16 * MT places, of the whole selection
  int tiles_per_block;
  int tiles_per_cta;
  int heads_per_cta;
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

// The scales of one row, one per unit, two to a word.
template <int UNITS>
struct UnitScales {
  uint32_t w[(UNITS + 1) / 2];
};

template <int UNITS, int PER>
__device__ __forceinline__ void spread(const uint32_t (&raw)[(UNITS + 1) / 2], UnitScales<UNITS>& s) {
  // unit u takes half u / PER of raw
#pragma unroll
  for (int i = 0; i < (UNITS + 1) / 2; ++i) {
    const int u0 = 2 * i / PER, u1 = (2 * i + 1) / PER;
    const uint32_t lo = u0 & 1 ? raw[u0 / 2] >> 16 : raw[u0 / 2] & 0xFFFFu;
    const uint32_t hi = u1 / 2 < (UNITS + 1) / 2
                            ? (u1 & 1 ? raw[u1 / 2] & 0xFFFF0000u : raw[u1 / 2] << 16)
                            : 0u;
    s.w[i] = lo | hi;
  }
}

// Loads the `groups` scales of a row and spreads them over its units (groups is the same for all
// threads, so the branches are uniform).
template <int UNITS>
__device__ __forceinline__ void load_scales(const __half* p, int groups, UnitScales<UNITS>& s) {
  constexpr int W = (UNITS + 1) / 2;
  uint32_t raw[W] = {};
  if (groups % 8 == 0) {
#pragma unroll
    for (int i = 0; i < W / 4; ++i)
      if (8 * i < groups) {
        const uint4 v = *reinterpret_cast<const uint4*>(p + 8 * i);
        raw[4 * i] = v.x, raw[4 * i + 1] = v.y, raw[4 * i + 2] = v.z, raw[4 * i + 3] = v.w;
      }
  } else if (groups == 4) {
    if constexpr (W >= 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      raw[0] = v.x, raw[1] = v.y;
    }
  } else if (groups % 2 == 0) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (2 * i < groups) raw[i] = reinterpret_cast<const uint32_t*>(p)[i];
  } else {
    const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (2 * i < groups) raw[i] = u[2 * i];
      if (2 * i + 1 < groups) raw[i] |= static_cast<uint32_t>(u[2 * i + 1]) << 16;
    }
  }
  const int per = UNITS / groups;
  if (per == 1) {
#pragma unroll
    for (int i = 0; i < W; ++i) s.w[i] = raw[i];
  } else if (per == 2) {
    spread<UNITS, 2>(raw, s);
  } else if (per == 3) {
    spread<UNITS, 3>(raw, s);
  } else if (per == 4) {
    spread<UNITS, 4>(raw, s);
  } else if (per == 8) {
    spread<UNITS, 8>(raw, s);
  } else {  // one group: 6 or 16 units
    spread<UNITS, 16>(raw, s);
  }
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
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if constexpr (kOwn == 8) {
          load_query8(a.query, a.dtype, at + u * UNIT + c * kOwn, q[u]);
        } else {
#pragma unroll
          for (int i = 0; i < kOwn; ++i) q[u][i] = load_query(a.query, a.dtype, at + u * UNIT + c * kOwn + i);
        }
#pragma unroll
        for (int i = 0; i < kOwn; ++i) top = fmaxf(top, fabsf(q[u][i]));
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

// What the weights kernels keep of a query row.
struct alignas(8) RowInfo {
  float factor, lse2;
};

// Places of a warp's tile: 32 where the query fragments come from shared memory (each load then
// feeds two MMAs) and both tiles' codes fit the registers.
constexpr int tile_rows(int d, int unit, int mode) {
  return mode != kStep && d <= 128 && unit == 32 ? 32 : 16;
}
constexpr int stages(int mode) { return mode == kStep ? 3 : 2; }
// Resident CTAs to leave registers for.
constexpr int resident(int d, bool lo, int mode) {
  return mode == kStep && d <= 128 && !lo ? 3 : (d == 256 && lo ? 1 : 2);
}

template <int BITS, int D, int UNIT, bool LO, int MODE>
__global__ void __launch_bounds__(kThreads, resident(D, LO, MODE)) weights_tc_kernel(const Job j) {
  using S = Shape<BITS, D, UNIT>;
  constexpr int kRows = tile_rows(D, UNIT, MODE), MT = kRows / 16, kDepth = stages(MODE);
  constexpr int kStage = kRows * S::kRowBytes;
  constexpr int kSteps = S::kPairs / 2;  // MMAs a unit
  extern __shared__ __align__(128) uint8_t smem[];
  // per warp: kDepth stages; then (not kStep) the row tiles' fragments, infos and visible counts
  const WeightsArgs& a = j.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = lane >> 2, c = lane & 3;
  const int heads = j.heads_per_cta, sub = warp / heads, subs = kWarps / heads;
  const int h = blockIdx.y * heads + warp % heads;
  const bool working = sub < subs;
  uint8_t* ring = smem + warp * kDepth * kStage;
  uint8_t* at = smem + kWarps * kDepth * kStage;
  using Frag = uint32_t[S::kPairs];
  Frag* frags = reinterpret_cast<Frag*>(at);  // [row_tiles][LO ? 2 : 1][units][32]
  constexpr int kFrags = (LO ? 2 : 1) * S::kUnits;  // of a row tile: the high parts, then the low
  constexpr int kTileFrags = kFrags * 32;
  RowInfo* infos = reinterpret_cast<RowInfo*>(frags + j.row_tiles * kTileFrags);
  int* seen = reinterpret_cast<int*>(infos + 8 * j.row_tiles);  // visible places of each row

  pdl_wait();
  pdl_launch();

  // ---- copies: this warp's tiles are first, first + subs, ... of the CTA's run
  const int run = blockIdx.x * j.tiles_per_cta;
  const int end = working ? min(j.total_tiles, run + j.tiles_per_cta) : 0;
  int next = run + sub;  // the next tile to copy
  int cached = -64, c_blk = -1, c_valid = 0;
  UnitScales<S::kUnits> scales[kDepth];
  int rows_of[kDepth];  // valid rows of the stage's tile
  float prev[kDepth];
  const auto issue = [&](int st) {
    rows_of[st] = 0;
    if (next < end) {
      const int slot = next / j.tiles_per_block, row0 = (next - slot * j.tiles_per_block) * kRows;
      if (slot < cached || slot >= cached + 32) {  // the warp's next 32 blocks, one per lane
        cached = slot;
        c_blk = -1;
        c_valid = 0;
        if (slot + lane < a.n_sel) {
          c_blk = a.table ? a.table[slot + lane] : slot + lane;
          if (c_blk < 0 || c_blk >= a.n_pool) {
            if (a.status) atomicOr(a.status, kDevBadBlockIndex);
            c_blk = -1;
          } else {
            c_valid = a.valid[c_blk];
            if ((c_valid < 0 || c_valid > a.bt) && a.status) atomicOr(a.status, kDevBadValidCount);
            c_valid = min(max(c_valid, 0), a.bt);
          }
        }
      }
      const int blk = __shfl_sync(0xffffffffu, c_blk, slot - cached);
      const int rows = min(kRows, __shfl_sync(0xffffffffu, c_valid, slot - cached) - row0);
      rows_of[st] = max(rows, 0);
      const long long tok = static_cast<long long>(blk) * a.bt + row0;
      const uint32_t dst = smem_addr(ring + st * kStage);
#pragma unroll
      for (int i = lane; i < kRows * S::kChunks; i += 32) {
        const int row = i / S::kChunks, q = i % S::kChunks;
        if (row < rows) {
          const uint8_t* src = a.kp + ((tok + row) * a.kvh + h) * S::kRowBytes + q * S::kChunk;
          const uint32_t to = dst + row * S::kRowBytes + (q ^ S::swizzle(row)) * S::kChunk;
          if constexpr (S::kChunk == 16) cp_async16(to, src, l2_evict_first());
          else cp_async8(to, src, l2_evict_first());
        }
      }
      const int srow = MT == 2 ? lane : lane & 15;
      if (srow < rows)
        load_scales<S::kUnits>(a.ks + ((tok + srow) * a.kvh + h) * (D / a.group), D / a.group,
                               scales[st]);
      else
        for (auto& w : scales[st].w) w = 0u;
      if constexpr (MODE != kLse) {
        const int orow = row0 + r + 8 * c;
        prev[st] = 0.f;
        if (c < 2 * MT && orow < a.bt && (a.previous || j.add)) {
          const long long place = static_cast<long long>(slot) * a.bt + orow;
          prev[st] = j.add ? a.out[h * a.out_stride + place] : a.previous[h * a.previous_stride + place];
        }
      }
    }
    cp_async_commit();
    next += subs;
  };
#pragma unroll
  for (int st = 0; st < kDepth - 1; ++st) issue(st);

  // ---- the query rows
  const int gqa = a.qh / a.kvh;
  QueryTile<D, UNIT, LO> own;  // kStep: this warp's head
  float factor[2], lse2[2];    // kStep: of columns 2c, 2c + 1
  int vis[2] = {0x7fffffff, 0x7fffffff};
  int all_see = 0x7fffffff;    // places below are seen by every row that sees anything
  if constexpr (MODE == kStep) {
    if (working) {
      own.load(j, h, 0, lane);
      float l2 = INFINITY;  // of row lane / 4, in the lanes c == 0
      for (int i = 0; i < 8; ++i) {
        const int row = j.row0 + i;
        if (row >= j.rows) break;
        const int t = row / gqa;
        const long long to = static_cast<long long>(t) * a.qh + h * gqa + row % gqa;
        float v;
        if (j.parts) {
          const float m = combine_parts(j, h, row, lane);
          if (blockIdx.x == 0 && sub == 0 && lane == 0) a.lse[to] = m * kLn2;
          v = m == -INFINITY ? INFINITY : m;
        } else {
          v = as_log2(a.lse_in[to]);
        }
        if (r == i) l2 = v;
        if (a.visible) {
          const int n = a.visible[t];
          if (2 * c == i) vis[0] = n;
          if (2 * c + 1 == i) vis[1] = n;
          if (n > 0) all_see = min(all_see, n);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        factor[i] = __shfl_sync(0xffffffffu, own.factor, 4 * (2 * c + i));
        lse2[i] = __shfl_sync(0xffffffffu, l2, 4 * (2 * c + i));
        if (vis[i] <= 0) lse2[i] = INFINITY;
      }
    }
  } else {
    const int h0 = blockIdx.y;  // one head a CTA
    for (int t = warp; t < j.row_tiles; t += kWarps) {
      QueryTile<D, UNIT, LO> q;
      q.load(j, h0, t, lane);
#pragma unroll
      for (int u = 0; u < kFrags; ++u)
#pragma unroll
        for (int p = 0; p < S::kPairs; ++p)
          frags[t * kTileFrags + u * 32 + lane][p] = q.b[u][p];
      if (c == 0) infos[8 * t + r].factor = q.factor;
    }
    for (int i = warp; i < 8 * j.row_tiles; i += kWarps) {
      const int row = j.row0 + i;
      int n = 0;
      float v = MODE == kLse ? 0.f : INFINITY;
      if (row < j.rows) {
        const int t = row / gqa;
        n = a.visible ? a.visible[t] : 0x7fffffff;
        if constexpr (MODE == kWindow) {
          const long long to = static_cast<long long>(t) * a.qh + h0 * gqa + row % gqa;
          if (j.parts) {
            const float m = combine_parts(j, h0, row, lane);
            if (blockIdx.x == 0 && lane == 0) a.lse[to] = m * kLn2;
            v = m == -INFINITY ? INFINITY : m;
          } else {
            v = as_log2(a.lse_in[to]);
          }
          if (n <= 0) v = INFINITY;
        }
      }
      if (lane == 0) {
        seen[i] = n;
        infos[i].lse2 = v;
      }
    }
    __syncthreads();
    for (int i = lane; i < 8 * j.row_tiles; i += 32)
      if (seen[i] > 0) all_see = min(all_see, seen[i]);
    all_see = __reduce_min_sync(0xffffffffu, all_see);
  }

  // ---- the tiles
  float run_m[MODE == kLse ? 2 * kLseTiles : 1], run_l[MODE == kLse ? 2 * kLseTiles : 1];
  if constexpr (MODE == kLse) {
#pragma unroll
    for (int i = 0; i < 2 * kLseTiles; ++i) run_m[i] = kLowest, run_l[i] = 0.f;
  }
  for (int tile = run + sub; tile < end;) {
#pragma unroll
    for (int st = 0; st < kDepth; ++st) {
      if (tile >= end) break;
      cp_async_wait<kDepth - 2>();
      __syncwarp();  // this tile's bytes are there; every lane is done with the tile before it
      issue((st + kDepth - 1) % kDepth);
      const int slot = tile / j.tiles_per_block, row0 = (tile - slot * j.tiles_per_block) * kRows;
      const int rows = rows_of[st];
      float sum[2 * MT] = {};
      if (rows > 0) {
        // K fragments of the tile: exact centred codes
        uint32_t k[MT][S::kUnits][S::kPairs][2];  // [..][pair][row r, row r + 8]
        const uint32_t src = smem_addr(ring + st * kStage);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if constexpr (BITS == 4 && UNIT == 32) {
            // ldmatrix: lanes 8 i .. 8 i + 7 give the rows of matrix i: rows 0-7, rows 8-15 of unit
            // u, then of unit u + 1
#pragma unroll
            for (int u = 0; u < S::kUnits; u += 2) {
              const int row = 16 * m + (lane & 15), q = min(u + (lane >> 4), S::kUnits - 1);
              uint32_t x[4];
              ldsm_x4(src + row * S::kRowBytes + (q ^ S::swizzle(row)) * 16, x[0], x[1], x[2], x[3]);
#pragma unroll
              for (int v = 0; v < 2; ++v)
                if (u + v < S::kUnits)
#pragma unroll
                  for (int half = 0; half < 2; ++half) {
                    uint32_t p[S::kPairs];
                    unpack<BITS, UNIT>(x[2 * v + half], p);
#pragma unroll
                    for (int i = 0; i < S::kPairs; ++i) k[m][u + v][i][half] = p[i];
                  }
            }
          } else {
            constexpr int kOwn = UNIT * BITS / 32;  // bytes a lane holds of a unit's row
#pragma unroll
            for (int u = 0; u < S::kUnits; ++u)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const int row = 16 * m + r + 8 * half, b = u * UNIT * BITS / 8 + c * kOwn;
                const uint8_t* from = ring + st * kStage + row * S::kRowBytes +
                                      ((b / S::kChunk) ^ S::swizzle(row)) * S::kChunk + b % S::kChunk;
                uint32_t x;
                if constexpr (kOwn == 1) x = *from;
                else x = *reinterpret_cast<const unsigned short*>(from);
                uint32_t p[S::kPairs];
                unpack<BITS, UNIT>(x, p);
#pragma unroll
                for (int i = 0; i < S::kPairs; ++i) k[m][u][i][half] = p[i];
              }
          }
        }
        // the rows' scales, in FP32: [m][half][unit]
        float sk[2 * MT][S::kUnits];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i)
#pragma unroll
          for (int w = 0; w < (S::kUnits + 1) / 2; ++w) {
            const uint32_t v = __shfl_sync(0xffffffffu, scales[st].w[w], r + 8 * i);
            const __half2 two = u32_as_h2(v);
            sk[i][2 * w] = __low2float(two);
            if (2 * w + 1 < S::kUnits) sk[i][2 * w + 1] = __high2float(two);
          }
        const int place0 = slot * a.bt + row0;
        const bool full = rows == kRows && place0 + kRows <= all_see;

        // scores less the log-sum-exps of one tile of 8 query rows, in the log2 domain, -inf where
        // masked (whatever the log-sum-exp): s[m][0..3] = rows r (columns 2c,
        // 2c + 1) and r + 8 of place tile m
        const auto scores = [&](const Frag (&b)[kFrags], RowInfo i0, RowInfo i1, int v0, int v1,
                                float (&s)[MT][4]) {
#pragma unroll
          for (int u = 0; u < S::kUnits; ++u) {
            const Frag& bh = b[u];
            const Frag& bl = b[LO ? S::kUnits + u : u];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int t = 0; t < kSteps; ++t) {
                mma_16816(acc, k[m][u][2 * t][0], k[m][u][2 * t][1], k[m][u][2 * t + 1][0],
                          k[m][u][2 * t + 1][1], bh[2 * t], bh[2 * t + 1]);
                if constexpr (LO)
                  mma_16816(acc, k[m][u][2 * t][0], k[m][u][2 * t][1], k[m][u][2 * t + 1][0],
                            k[m][u][2 * t + 1][1], bl[2 * t], bl[2 * t + 1]);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float scale = sk[2 * m + (i >> 1)][u];
                s[m][i] = u == 0 ? acc[i] * scale : fmaf(acc[i], scale, s[m][i]);
              }
            }
          }
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              s[m][i] = i & 1 ? fmaf(s[m][i], i1.factor, -i1.lse2) : fmaf(s[m][i], i0.factor, -i0.lse2);
              if (!full) {
                const int row = 16 * m + r + 8 * (i >> 1);
                if (row >= rows || place0 + row >= (i & 1 ? v1 : v0)) s[m][i] = -INFINITY;
              }
            }
        };

        if constexpr (MODE == kStep) {
          float s[MT][4];
          scores(own.b, {factor[0], lse2[0]}, {factor[1], lse2[1]}, vis[0], vis[1], s);
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              sum[2 * m + i] = fast_exp2(s[m][2 * i]) + fast_exp2(s[m][2 * i + 1]);
        } else if constexpr (MODE == kWindow) {
          for (int t = 0; t < j.row_tiles; ++t) {
            const float4 info = *reinterpret_cast<const float4*>(infos + 8 * t + 2 * c);
            int2 v = make_int2(0x7fffffff, 0x7fffffff);
            if (!full) v = *reinterpret_cast<const int2*>(seen + 8 * t + 2 * c);
            Frag b[kFrags];
#pragma unroll
            for (int u = 0; u < kFrags; ++u) load_fragment(frags[t * kTileFrags + u * 32 + lane], b[u]);
            float s[MT][4];
            scores(b, {info.x, info.y}, {info.z, info.w}, v.x, v.y, s);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int i = 0; i < 2; ++i)
                sum[2 * m + i] += fast_exp2(s[m][2 * i]) + fast_exp2(s[m][2 * i + 1]);
          }
        } else {
#pragma unroll
          for (int t = 0; t < kLseTiles; ++t) {
            if (t >= j.row_tiles) break;
            const float4 info = *reinterpret_cast<const float4*>(infos + 8 * t + 2 * c);
            int2 v = make_int2(0x7fffffff, 0x7fffffff);
            if (!full) v = *reinterpret_cast<const int2*>(seen + 8 * t + 2 * c);
            Frag b[kFrags];
#pragma unroll
            for (int u = 0; u < kFrags; ++u) load_fragment(frags[t * kTileFrags + u * 32 + lane], b[u]);
            float s[MT][4];
            scores(b, {info.x, info.y}, {info.z, info.w}, v.x, v.y, s);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float top = fmaxf(s[0][i], s[0][2 + i]);
#pragma unroll
              for (int m = 1; m < MT; ++m) top = fmaxf(top, fmaxf(s[m][i], s[m][2 + i]));
              float& rm = run_m[2 * t + i];
              float& rl = run_l[2 * t + i];
              if (top > rm + 8.f) {  // the running max moves only past 2^8: terms stay finite
                rl *= fast_exp2(rm - top);
                rm = top;
              }
#pragma unroll
              for (int m = 0; m < MT; ++m) rl += fast_exp2(s[m][i] - rm) + fast_exp2(s[m][2 + i] - rm);
            }
          }
        }
      }
      if constexpr (MODE != kLse) {
        // sum over the tile's query rows: lane c of a row group ends with place r + 8 c
        float mine;
        if constexpr (MT == 1) {
          const float give = c & 1 ? sum[0] : sum[1];
          mine = (c & 1 ? sum[1] : sum[0]) + __shfl_xor_sync(0xffffffffu, give, 1);
          mine += __shfl_xor_sync(0xffffffffu, mine, 2);
        } else {
          const float g0 = c & 1 ? sum[0] : sum[1], g1 = c & 1 ? sum[2] : sum[3];
          const float k0 = (c & 1 ? sum[1] : sum[0]) + __shfl_xor_sync(0xffffffffu, g0, 1);
          const float k1 = (c & 1 ? sum[3] : sum[2]) + __shfl_xor_sync(0xffffffffu, g1, 1);
          mine = (c & 2 ? k1 : k0) + __shfl_xor_sync(0xffffffffu, c & 2 ? k0 : k1, 2);
        }
        const int orow = row0 + r + 8 * c;
        if (c < 2 * MT && orow < a.bt)
          a.out[h * a.out_stride + static_cast<long long>(slot) * a.bt + orow] = prev[st] + mine;
      }
      tile += subs;
    }
  }
  cp_async_wait<0>();

  if constexpr (MODE == kLse) {
    // parts of the CTA's run: over the 8 row lanes of a column, then over the warps
    __syncthreads();  // the ring is free
    float2* mine = reinterpret_cast<float2*>(smem) + warp * 8 * kLseTiles;
#pragma unroll
    for (int i = 0; i < 2 * kLseTiles; ++i) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, run_m[i], o);
        const float l2 = __shfl_xor_sync(0xffffffffu, run_l[i], o);
        const float top = fmaxf(run_m[i], m2);
        run_l[i] = run_l[i] * fast_exp2(run_m[i] - top) + l2 * fast_exp2(m2 - top);
        run_m[i] = top;
      }
      if (r == 0) mine[(i >> 1) * 8 + 2 * c + (i & 1)] = make_float2(run_m[i], run_l[i]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * j.row_tiles && j.row0 + i < j.rows; i += kThreads) {
      float m = kLowest, l = 0.f;
      for (int w = 0; w < kWarps; ++w) {
        const float2 v = reinterpret_cast<const float2*>(smem)[w * 8 * kLseTiles + i];
        const float top = fmaxf(m, v.x);
        l = l * fast_exp2(m - top) + v.y * fast_exp2(v.x - top);
        m = top;
      }
      if (seen[i] <= 0) m = kLowest, l = 0.f;
      reinterpret_cast<float2*>(a.scratch)[(static_cast<long long>(blockIdx.y) * j.rows + j.row0 + i) *
                                               j.parts + blockIdx.x] = make_float2(m, l);
    }
  }
}

// Grid of a launch over `total` tiles and kvh heads, `heads` of them a CTA: as many CTAs as are
// resident at once, each with a contiguous run of tiles.
inline int grid_x(int total, int kvh, int heads, int ctas) {
  const int subs = kWarps / heads, ys = kvh / heads;
  const int most = (total + subs - 1) / subs, want = 148 * ctas / ys;
  return want < 1 ? 1 : (want < most ? want : most);
}

template <int D, int UNIT, int MODE>
int tiles_per_block(int bt) {
  return (bt + tile_rows(D, UNIT, MODE) - 1) / tile_rows(D, UNIT, MODE);
}

// Parts per query row of the log-sum-exp pass.
template <int D, int UNIT, bool LO>
int lse_parts(int n_sel, int bt, int kvh) {
  return grid_x(n_sel * tiles_per_block<D, UNIT, kLse>(bt), kvh, 1, resident(D, LO, kLse));
}

template <int BITS, int D, int UNIT, bool LO, int MODE>
cudaError_t launch_mode(Job j, cudaStream_t s) {
  using S = Shape<BITS, D, UNIT>;
  const auto kernel = weights_tc_kernel<BITS, D, UNIT, LO, MODE>;
  const WeightsArgs& a = j.a;
  j.tiles_per_block = tiles_per_block<D, UNIT, MODE>(a.bt);
  j.total_tiles = a.n_sel * j.tiles_per_block;
  j.heads_per_cta = 1;
  if (MODE == kStep)
    for (int i = 2; i <= kWarps; ++i)
      if (a.kvh % i == 0) j.heads_per_cta = i;
  const int gx = grid_x(j.total_tiles, a.kvh, j.heads_per_cta, resident(D, LO, MODE));
  j.tiles_per_cta = (j.total_tiles + gx - 1) / gx;
  constexpr size_t ring = static_cast<size_t>(kWarps) * stages(MODE) * tile_rows(D, UNIT, MODE) * S::kRowBytes;
  constexpr size_t row_tile = (LO ? 2 : 1) * S::kUnits * 32 * S::kPairs * 4 + 8 * (sizeof(RowInfo) + sizeof(int));
  static_assert(MODE != kLse || ring >= kWarps * 8 * kLseTiles * sizeof(float2), "the parts use the ring");
  const int all = (j.rows + 7) / 8;
  // kWindow keeps as many row tiles as leave two CTAs' shared memory on an SM, or one's when that
  // saves a pass over the keys
  constexpr int two = static_cast<int>((110 * 1024 - ring) / row_tile), one = static_cast<int>((220 * 1024 - ring) / row_tile);
  const int most = MODE == kStep ? 1 : MODE == kLse ? kLseTiles : all <= two ? two : one;
  for (j.row0 = 0; j.row0 < j.rows; j.row0 += 8 * j.row_tiles) {
    const int left = all - j.row0 / 8;
    j.row_tiles = left < most ? left : most;
    j.add = j.row0 > 0;
    const size_t smem = ring + (MODE == kStep ? 0 : j.row_tiles * row_tile);
    cudaError_t e = cudaSuccess;
    if (smem > 48 * 1024)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e == cudaSuccess)
      e = launch_pdl(kernel, dim3(gx, a.kvh / j.heads_per_cta), kThreads, smem, s, j);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <int BITS, int D, int UNIT, bool LO>
cudaError_t launch_shape(const WeightsArgs& a, cudaStream_t s) {
  Job j{};
  j.a = a;
  j.rows = a.queries * (a.qh / a.kvh);
  if (!a.lse_in) {
    j.parts = lse_parts<D, UNIT, LO>(a.n_sel, a.bt, a.kvh);
    const cudaError_t e = launch_mode<BITS, D, UNIT, LO, kLse>(j, s);
    if (e != cudaSuccess) return e;
  }
  if (j.rows <= 8) return launch_mode<BITS, D, UNIT, LO, kStep>(j, s);
  return launch_mode<BITS, D, UNIT, LO, kWindow>(j, s);
}

template <int D>
cudaError_t launch(const WeightsArgs& a, cudaStream_t s) {
  const bool lo = a.dtype == kQF32 || a.dtype == kQF64;
  if (a.bits == 4) {
    if (a.group % 32 == 0) return lo ? launch_shape<4, D, 32, true>(a, s) : launch_shape<4, D, 32, false>(a, s);
    return lo ? launch_shape<4, D, 16, true>(a, s) : launch_shape<4, D, 16, false>(a, s);
  }
  if (a.group % 32 == 0) return lo ? launch_shape<2, D, 32, true>(a, s) : launch_shape<2, D, 32, false>(a, s);
  return lo ? launch_shape<2, D, 16, true>(a, s) : launch_shape<2, D, 16, false>(a, s);
}

}  // namespace weights_tc

// Launchers, one translation unit per head_dim.
cudaError_t launch_weights_tc_64(const WeightsArgs& a, cudaStream_t s);
cudaError_t launch_weights_tc_96(const WeightsArgs& a, cudaStream_t s);
cudaError_t launch_weights_tc_128(const WeightsArgs& a, cudaStream_t s);
cudaError_t launch_weights_tc_256(const WeightsArgs& a, cudaStream_t s);
}  // namespace kvb
