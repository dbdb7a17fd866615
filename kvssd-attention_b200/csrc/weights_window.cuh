// Attention weights of 9 to 32 query rows a KV head (of more where the tcgen05 kernel's shared memory does
// not suffice), and the log-sum-exp pass of up to 32.
//
// A warp unpacks a tile's keys into registers once and goes over the query rows 8 at a time, their
// fragments in shared memory: each load of a fragment feeds the MMAs of all of the tile's places. Bound by
// the instructions of a tile of 8 rows (MMAs, scales, exponentials and masks beside one another):
// 65536 tokens x 8 heads x 128 INT4, both passes, 16 rows 52 us, 32 rows 69 us.
#pragma once

#include "weights_tc.cuh"

namespace kvb {
namespace weights_tc {

// Places of a warp's tile: 32 where both halves' codes fit the registers (each load of a query
// fragment then feeds two MMAs).
constexpr int tile_rows(int d, int unit) { return d <= 128 && unit == 32 ? 32 : 16; }
constexpr int kStages = 2;
// Resident CTAs to leave registers for. (Units of 16 dims at head_dim 256 spill about 0.5 KB a thread at two.)
constexpr int resident(int d, bool lo) { return d == 256 && lo ? 1 : 2; }

template <int BITS, int D, int UNIT, bool LO, int MODE>
__global__ void __launch_bounds__(kThreads, resident(D, LO)) weights_tc_kernel(const Job j) {
  using S = Shape<BITS, D, UNIT>;
  constexpr int kRows = tile_rows(D, UNIT), MT = kRows / 16, kDepth = kStages;
  constexpr int kStage = kRows * S::kRowBytes;
  constexpr int kSteps = S::kPairs / 2;  // MMAs a unit
  extern __shared__ __align__(128) uint8_t smem[];
  // per warp: kDepth stages; then the row tiles' fragments, infos and visible counts
  const WeightsArgs& a = j.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = lane >> 2, c = lane & 3;
  const int h = blockIdx.y;
  const int groups = D / a.group;
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

  // ---- copies: this warp's tiles are first, first + kWarps, ... of the CTA's run
  const int run = blockIdx.x * j.tiles_per_cta;
  const int end = min(j.total_tiles, run + j.tiles_per_cta);
  int next = run + warp;  // the next tile to copy
  int cached = -64, c_blk = -1, c_valid = 0;
  RowScales<S::kUnits> scales[kDepth];
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
#pragma unroll
      for (int i = 0; i < (S::kUnits + 1) / 2; ++i) scales[st].w[i] = 0u;
      if (srow < rows)
        load_scales<S::kUnits>(a.ks + ((tok + srow) * a.kvh + h) * groups, groups, scales[st]);
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
    next += kWarps;
  };
#pragma unroll
  for (int st = 0; st < kDepth - 1; ++st) issue(st);

  // ---- the query rows
  const int gqa = a.qh / a.kvh;
  int all_see = 0x7fffffff;    // places below are seen by every row that sees anything
  for (int t = warp; t < j.row_tiles; t += kWarps) {
    QueryTile<D, UNIT, LO> q;
    q.load(j, h, t, lane);
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
        const long long to = static_cast<long long>(t) * a.qh + h * gqa + row % gqa;
        if (j.parts) {
          const float m = combine_parts(j, h, row, lane);
          if (blockIdx.x == 0 && lane == 0) a.lse[to] = m * kLn2;
          v = m == -INFINITY ? INFINITY : m;
        } else {
          v = as_log2(a.lse_in[to]);
        }
        if (n <= 0) v = INFINITY;
        if (v == INFINITY) n = 0;  // adds nothing, whatever a key's scale
      }
    }
    if (lane == 0) {
      seen[i] = n;
      infos[i].lse2 = v;
    }
  }
  __syncthreads();
  bool any = false;
  for (int i = lane; i < 8 * j.row_tiles; i += 32)
    if (seen[i] > 0) all_see = min(all_see, seen[i]), any = true;
  all_see = __reduce_min_sync(0xffffffffu, all_see);
  if (!__any_sync(0xffffffffu, any)) all_see = 0;  // nothing is seen: mask every tile

  // ---- the tiles
  float run_m[MODE == kLse ? 2 * kLseTiles : 1], run_l[MODE == kLse ? 2 * kLseTiles : 1];
  if constexpr (MODE == kLse) {
#pragma unroll
    for (int i = 0; i < 2 * kLseTiles; ++i) run_m[i] = kLowest, run_l[i] = 0.f;
  }
  for (int tile = run + warp; tile < end;) {
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
        const RowScales<S::kUnits> mine = spread<S::kUnits>(scales[st], groups);
        float sk[2 * MT][S::kUnits];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i)
#pragma unroll
          for (int w = 0; w < (S::kUnits + 1) / 2; ++w) {
            const uint32_t v = __shfl_sync(0xffffffffu, mine.w[w], r + 8 * i);
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

        if constexpr (MODE == kWindow) {
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
      tile += kWarps;
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

template <int BITS, int D, int UNIT, bool LO, int MODE>
cudaError_t launch_mode(Job j, cudaStream_t s) {
  using S = Shape<BITS, D, UNIT>;
  const auto kernel = weights_tc_kernel<BITS, D, UNIT, LO, MODE>;
  const WeightsArgs& a = j.a;
  const int gx = grid_x(j.total_tiles, a.kvh, 1, kWarps, resident(D, LO));
  j.tiles_per_cta = (j.total_tiles + gx - 1) / gx;
  constexpr size_t ring = static_cast<size_t>(kWarps) * kStages * tile_rows(D, UNIT) * S::kRowBytes;
  constexpr size_t row_tile = (LO ? 2 : 1) * S::kUnits * 32 * S::kPairs * 4 + 8 * (sizeof(RowInfo) + sizeof(int));
  static_assert(MODE != kLse || ring >= kWarps * 8 * kLseTiles * sizeof(float2), "the parts use the ring");
  const int all = (j.rows + 7) / 8;
  // kWindow keeps as many row tiles as leave two CTAs' shared memory on an SM, or one's when that
  // saves a pass over the keys
  constexpr int two = static_cast<int>((110 * 1024 - ring) / row_tile), one = static_cast<int>((220 * 1024 - ring) / row_tile);
  const int most = MODE == kLse ? kLseTiles : all <= two ? two : one;
  for (j.row0 = 0; j.row0 < j.rows; j.row0 += 8 * j.row_tiles) {
    const int left = all - j.row0 / 8;
    j.row_tiles = left < most ? left : most;
    j.add = j.row0 > 0;
    const size_t smem = ring + j.row_tiles * row_tile;
    cudaError_t e = cudaSuccess;
    if (smem > 48 * 1024)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e == cudaSuccess) e = launch_pdl(kernel, dim3(gx, a.kvh), kThreads, smem, s, j);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace weights_tc
}  // namespace kvb
