// Attention weights of at most 8 query rows a KV head (a decode step): one pass over the keys.
//
// Bound by HBM: per place and head the codes and scales (72 bytes at INT4, group 32, head_dim 128) and
// 8 bytes of running sums. A warp keeps its head's query fragments in registers and streams tiles of
// 32 (or 16) places through a private cp.async ring; what it spends per tile has to stay under the
// copies' time, so INT4 codes are not centred: they enter the MMAs as FP16 subnormals n 2^-24 (a mask
// per pair; the slots whose bits lie higher in the lane have their queries divided by that power of
// two), and the accumulator starts at -8 2^-24 sum q, which is constant. The MMAs' FP32 sums then
// round at the size of that start, which is the size of the codes' own sum. INT2 codes are mostly
// zero, their sums far below such a start, so they are centred first (half as many bytes to unpack).
//
// One step of 8 KV heads x 4 query heads x 128: 131072 tokens INT4 21.4 us, 0.60 of the measured copy
// rate (84 MB; about 5 us are the start, the rest runs at 0.78 of that rate, bound by issuing: 355
// instructions a 32-place tile, the start's included, in half of all issue slots at 16 warps an SM); INT2
// 22.3 us (398 instructions); 8192 tokens 6.2 us, all of it start. FP32 queries 29 us. Tiles of 16
// places with three or four CTAs an SM took 28 to 36 us.
#pragma once

#include "weights_tc.cuh"

namespace kvb {
namespace weights_tc {

constexpr int kStepStages = 3;
constexpr float kTiny = 5.9604644775390625e-8f;  // 2^-24, FP16's smallest subnormal
constexpr int step_rows(int d, int unit, bool lo) { return d <= 128 && unit == 32 && !lo ? 32 : 16; }
// Resident CTAs to leave registers for. Units of 16 dims at head_dim 256 spill about 0.5 KB a thread at two
// (131072 places x 4 heads INT4 in groups of 16: 57 us).
constexpr int step_resident(int d, bool lo) { return d == 256 && lo ? 1 : 2; }

// Codes of one lane, row and unit: INT4 as pairs n 2^-24 2^step_shift(p), INT2 centred.
template <int BITS, int UNIT>
__device__ __forceinline__ void unpack_step(uint32_t x, uint32_t (&p)[UNIT / 8]) {
  if constexpr (BITS == 2) {
    unpack<BITS, UNIT>(x, p);
  } else if constexpr (UNIT == 32) {
    p[0] = x & 0x000F000Fu;
    p[1] = x & 0x00F000F0u;
    p[2] = (x >> 8) & 0x000F000Fu;
    p[3] = (x >> 8) & 0x00F000F0u;
  } else {
    const uint32_t y = __byte_perm(x, 0, 0x4140);
    p[0] = y & 0x000F000Fu;
    p[1] = y & 0x00F000F0u;
  }
}
constexpr int step_shift(int p) { return 4 * (p & 1); }

// What a CTA's warps need to know of a tile, looked up once by all threads before they start.
struct alignas(16) Tile {
  long long row;  // its first token's row of KV head 0, in (token, head) rows of the pool
  int place;
  int rows;       // valid rows | rows of the block from here on << 16
};
constexpr int kMostTiles = 1024;  // a CTA

template <int BITS, int D, int UNIT, bool LO, bool GROUPED>
__global__ void __launch_bounds__(kThreads, step_resident(D, LO)) weights_step_kernel(const Job j) {
  using S = Shape<BITS, D, UNIT>;
  constexpr int kRows = step_rows(D, UNIT, LO), MT = kRows / 16;
  constexpr int kStage = kRows * S::kRowBytes, kSteps = S::kPairs / 2;
  constexpr int kScaleWords = (S::kUnits + 1) / 2;
  constexpr int kCopies = (kRows * S::kChunks + 31) / 32;  // a lane and tile
  extern __shared__ __align__(128) uint8_t smem[];
  const WeightsArgs& a = j.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = lane >> 2, c = lane & 3;
  const int heads = j.heads_per_cta, sub = warp / heads, subs = kWarps / heads;
  const int h = blockIdx.y * heads + warp % heads;
  // one scale per unit, or `groups` of them a row
  const int groups = GROUPED ? D / a.group : S::kUnits;
  const int run = blockIdx.x * j.tiles_per_cta;
  const int tiles = min(j.total_tiles - run, j.tiles_per_cta);  // of the CTA: every thread looks some up
  // of this warp; none for a warp left over where the heads do not divide the warps
  const int count = sub < subs && tiles > sub ? (tiles - sub + subs - 1) / subs : 0;
  Tile* tile_of = reinterpret_cast<Tile*>(smem);
  uint8_t* ring = smem + j.tiles_per_cta * sizeof(Tile) + warp * kStepStages * kStage;
  const uint32_t ring_at = smem_addr(ring);

  pdl_wait();
  pdl_launch();
  for (int i = threadIdx.x; i < tiles; i += kThreads) {
    const int slot = (run + i) / j.tiles_per_block, row0 = (run + i - slot * j.tiles_per_block) * kRows;
    int blk = a.table ? a.table[slot] : slot, valid = 0;
    if (blk < 0 || blk >= a.n_pool) {
      if (a.status) atomicOr(a.status, kDevBadBlockIndex);
      blk = 0;
    } else {
      valid = a.valid[blk];
      if ((valid < 0 || valid > a.bt) && a.status) atomicOr(a.status, kDevBadValidCount);
      valid = min(valid, a.bt);
    }
    tile_of[i] = {(static_cast<long long>(blk) * a.bt + row0) * a.kvh, slot * a.bt + row0,
                  max(0, min(kRows, valid - row0)) | min(kRows, a.bt - row0) << 16};
  }
  __syncthreads();

  // ---- copies of the warp's tiles: sub, sub + subs, ... of the CTA's run
  const uint64_t policy = l2_evict_first();
  RowScales<S::kUnits> scales[kStepStages];
  float prev[kStepStages];
  const int token_bytes = a.kvh * S::kRowBytes;
  const uint8_t* codes = a.kp + h * S::kRowBytes;
  const __half* rows_scales = a.ks + (static_cast<long long>(lane % kRows) * a.kvh + h) * groups;
  const int out_row = r + 8 * c;  // the place of a tile whose sum this lane ends with
  const float* before = a.previous ? a.previous + h * a.previous_stride + out_row : nullptr;
  float* sums = a.out + h * a.out_stride + out_row;
  const auto issue = [&](int st, int i) {
    if (i < count) {
      const Tile t = tile_of[sub + i * subs];
      const int rows = t.rows & 0xFFFF;
      const uint8_t* from = codes + t.row * S::kRowBytes;
#pragma unroll
      for (int k = 0; k < kCopies; ++k) {
        const int at = lane + 32 * k, row = at / S::kChunks, q = at % S::kChunks;
        const uint32_t to = ring_at + st * kStage + row * S::kRowBytes + (q ^ S::swizzle(row)) * S::kChunk;
        if (row < rows) {
          const uint8_t* src = from + (static_cast<long long>(row) * token_bytes + q * S::kChunk);
          if constexpr (S::kChunk == 16) cp_async16(to, src, policy);
          else cp_async8(to, src, policy);
        }
      }
#pragma unroll
      for (int w = 0; w < kScaleWords; ++w) scales[st].w[w] = 0u;
      if (lane % kRows < rows) load_scales<S::kUnits>(rows_scales + t.row * groups, groups, scales[st]);
      prev[st] = 0.f;
      if (before && c < 2 * MT && out_row < t.rows >> 16) prev[st] = before[t.place];
    }
    cp_async_commit();
  };
#pragma unroll
  for (int st = 0; st < kStepStages - 1; ++st) issue(st, st);

  // ---- the query rows of the warp's head
  QueryTile<D, UNIT, LO> q;
  float offset[S::kUnits][2] = {};  // the accumulators' start, of columns 2c, 2c + 1
  RowInfo info[2];
  int vis[2] = {0, 0};
  int all_see = 0;  // places below are seen by every row that sees anything
  if (count > 0) {
    q.load(j, h, 0, lane);
    if constexpr (BITS == 4) {
#pragma unroll
      for (int u = 0; u < S::kUnits; ++u) {
        float sum = 0.f;
#pragma unroll
        for (int p = 0; p < S::kPairs; ++p)
#pragma unroll
          for (int part = 0; part < (LO ? 2 : 1); ++part) {
            uint32_t& b = q.b[part * S::kUnits + u][p];
            const __half2 v = u32_as_h2(b);
            sum += __low2float(v) + __high2float(v);
            const float down = 1.f / static_cast<float>(1 << step_shift(p));
            b = h2_as_u32(__hmul2(v, __float2half2_rn(down)));
          }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          offset[u][i] = -8.f * kTiny * __shfl_sync(0xffffffffu, sum, 4 * (2 * c + i));
      }
    }
    const int gqa = a.qh / a.kvh;
    float l2 = INFINITY;  // lane i: of row i
    int see = 0;
    if (lane < j.rows) {
      see = a.visible ? max(a.visible[lane / gqa], 0) : 0x7fffffff;
      if (!j.parts)
        l2 = as_log2(a.lse_in[static_cast<long long>(lane / gqa) * a.qh + h * gqa + lane % gqa]);
    }
    if (j.parts) {
      for (int i = 0; i < j.rows; ++i) {
        const float m = combine_parts(j, h, i, lane);
        if (lane == i) l2 = m == -INFINITY ? INFINITY : m;
        if (blockIdx.x == 0 && sub == 0 && lane == 0)
          a.lse[static_cast<long long>(i / gqa) * a.qh + h * gqa + i % gqa] = m * kLn2;
      }
    }
    if (see <= 0) l2 = INFINITY;
    if (l2 == INFINITY) see = 0;  // adds nothing, whatever a key's scale
    all_see = __reduce_min_sync(0xffffffffu, see > 0 ? see : 0x7fffffff);
    if (!__any_sync(0xffffffffu, see > 0)) all_see = 0;  // nothing is seen: mask every tile
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      info[i].factor = __shfl_sync(0xffffffffu, q.factor, 4 * (2 * c + i)) * (BITS == 4 ? 1.f / kTiny : 1.f);
      info[i].lse2 = __shfl_sync(0xffffffffu, l2, 2 * c + i);
      vis[i] = __shfl_sync(0xffffffffu, see, 2 * c + i);
    }
  }

  // ---- the tiles
  // byte of the tile this lane's loads start at: ldmatrix rows (lane & 15) of the unit pair's chunk
  // lane >> 4, or this lane's bytes of row r
  const uint32_t own = BITS == 4 && UNIT == 32
                           ? (lane & 15) * S::kRowBytes
                           : r * S::kRowBytes;
  for (int first = 0; first < count; first += kStepStages) {
#pragma unroll
    for (int st = 0; st < kStepStages; ++st) {
      if (first + st >= count) break;
      cp_async_wait<kStepStages - 2>();
      __syncwarp();  // this tile's bytes are there; every lane is done with the tile before it
      issue((st + kStepStages - 1) % kStepStages, first + st + kStepStages - 1);
      const Tile t = tile_of[sub + (first + st) * subs];
      const int rows = t.rows & 0xFFFF;
      float sum[2 * MT] = {};
      if (rows > 0) {
        uint32_t raw[MT][S::kUnits][2];  // this lane's bytes of rows r and r + 8
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint32_t tile = st * kStage + 16 * m * S::kRowBytes;
          if constexpr (BITS == 4 && UNIT == 32) {
#pragma unroll
            for (int u = 0; u < S::kUnits; u += 2) {
              const int chunk = min(u + (lane >> 4), S::kUnits - 1) ^ S::swizzle(lane & 15);
              uint32_t x[4];
              ldsm_x4(ring_at + tile + own + chunk * 16, x[0], x[1], x[2], x[3]);
              raw[m][u][0] = x[0], raw[m][u][1] = x[1];
              if (u + 1 < S::kUnits) raw[m][u + 1][0] = x[2], raw[m][u + 1][1] = x[3];
            }
          } else {
            constexpr int kOwn = UNIT * BITS / 32;  // bytes a lane holds of a unit's row
#pragma unroll
            for (int u = 0; u < S::kUnits; ++u)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const int b = u * UNIT * BITS / 8 + c * kOwn;
                const uint8_t* from = ring + tile + own + 8 * half * S::kRowBytes +
                                      ((b / S::kChunk) ^ S::swizzle(r + 8 * half)) * S::kChunk + b % S::kChunk;
                if constexpr (kOwn == 1) raw[m][u][half] = *from;
                else raw[m][u][half] = *reinterpret_cast<const unsigned short*>(from);
              }
          }
        }
        const RowScales<S::kUnits> mine = GROUPED ? spread<S::kUnits>(scales[st], groups) : scales[st];
        float s[MT][4];
#pragma unroll
        for (int w = 0; w < kScaleWords; ++w) {
          float sk[2 * MT][2];  // of units 2w, 2w + 1 in the rows r + 8 i
#pragma unroll
          for (int i = 0; i < 2 * MT; ++i) {
            const __half2 two = u32_as_h2(__shfl_sync(0xffffffffu, mine.w[w], r + 8 * i));
            sk[i][0] = __low2float(two);
            sk[i][1] = __high2float(two);
          }
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const int u = 2 * w + v;
            if (u >= S::kUnits) continue;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              uint32_t k0[S::kPairs], k1[S::kPairs];
              unpack_step<BITS, UNIT>(raw[m][u][0], k0);
              unpack_step<BITS, UNIT>(raw[m][u][1], k1);
              float acc[4];
#pragma unroll
              for (int n = 0; n < kSteps; ++n) {
                if (n == 0)
                  mma_16816_from(acc, offset[u][0], offset[u][1], k0[0], k1[0], k0[1], k1[1],
                                 q.b[u][0], q.b[u][1]);
                else
                  mma_16816(acc, k0[2 * n], k1[2 * n], k0[2 * n + 1], k1[2 * n + 1], q.b[u][2 * n],
                            q.b[u][2 * n + 1]);
                if constexpr (LO)
                  mma_16816(acc, k0[2 * n], k1[2 * n], k0[2 * n + 1], k1[2 * n + 1],
                            q.b[S::kUnits + u][2 * n], q.b[S::kUnits + u][2 * n + 1]);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float scale = sk[2 * m + (i >> 1)][v];
                s[m][i] = u == 0 ? acc[i] * scale : fmaf(acc[i], scale, s[m][i]);
              }
            }
          }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[m][i] = fmaf(s[m][i], info[i & 1].factor, -info[i & 1].lse2);
        if (rows < kRows || t.place + kRows > all_see) {
          const int seen0 = min(rows, vis[0] - t.place), seen1 = min(rows, vis[1] - t.place);
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (16 * m + r + 8 * (i >> 1) >= (i & 1 ? seen1 : seen0)) s[m][i] = -INFINITY;
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            sum[2 * m + i] = fast_exp2(s[m][2 * i]) + fast_exp2(s[m][2 * i + 1]);
      }
      // sum over the columns: lane c of a row group ends with place r + 8 c
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
      if (c < 2 * MT && out_row < t.rows >> 16) sums[t.place] = prev[st] + mine;
    }
  }
  cp_async_wait<0>();
}

template <int BITS, int D, int UNIT, bool LO>
cudaError_t launch_step(Job j, cudaStream_t s) {
  using S = Shape<BITS, D, UNIT>;
  const WeightsArgs& a = j.a;
  constexpr int rows = step_rows(D, UNIT, LO);
  j.tiles_per_block = (a.bt + rows - 1) / rows;
  j.total_tiles = a.n_sel * j.tiles_per_block;
  j.heads_per_cta = 1;
  for (int i = 2; i <= kWarps; ++i)
    if (a.kvh % i == 0) j.heads_per_cta = i;
  const int gx = grid_x(j.total_tiles, a.kvh, j.heads_per_cta, kWarps, step_resident(D, LO));
  j.tiles_per_cta = (j.total_tiles + gx - 1) / gx;
  if (j.tiles_per_cta > kMostTiles) j.tiles_per_cta = kMostTiles;  // a very long cache: more CTAs
  const int ctas = (j.total_tiles + j.tiles_per_cta - 1) / j.tiles_per_cta;
  const auto kernel = a.group == UNIT ? weights_step_kernel<BITS, D, UNIT, LO, false>
                                      : weights_step_kernel<BITS, D, UNIT, LO, true>;
  const size_t smem = j.tiles_per_cta * sizeof(Tile) + static_cast<size_t>(kWarps) * kStepStages * rows * S::kRowBytes;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(kernel, dim3(ctas, a.kvh / j.heads_per_cta), kThreads, smem, s, j);
}

}  // namespace weights_tc
}  // namespace kvb
