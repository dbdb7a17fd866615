// Attention weights of many query rows a KV head (a prompt's window) on the 5th-generation tensor cores:
// head_dim 64, 96, 128 and 256, scale groups of whole 16 dims.
//
// Math. A tile is 128 places by up to 128 query rows. The places' keys are dequantized into shared memory
// as FP16: a centred INT2 code times its FP16 scale is exact in FP16; an INT4 one has up to 14 bits and
// goes in as two FP16 terms, hi = RN(code * scale) and lo = code * scale - hi, which is exact. Queries
// are FP16 (FP32 and FP64 ones a high and a low part), each row brought to the top of FP16's range by a
// power of two (what that rounds is said in weights_tc.cuh). Of two keys' terms and two queries' the product
// of the low ones, 2^-22 of the whole, is left out. No scale is applied behind tcgen05.mma's FP32 sums.
// Scales so large that a product leaves FP16's range (above 8188, or 32752 at INT2) are divided by 16
// for the whole tile, whose scores are multiplied by 16 again (scales below 2^-10 beside them are
// rounded to FP16's subnormals then: an element of such a key is off by up to 2^-18, where one of the large
// scale's is a multiple of 2^13).
//
// Two passes: the log-sum-exps put the queries on the accumulator's lanes and the places on its columns
// (a thread keeps the running max and sum of its query row), the weights the other way round (a thread
// sums over its place's columns), so neither reduces across lanes. Bound by the exponentials: two per
// score, 16 a clock and SM -- 1024 clocks a tile and pass, beside 512 (INT2) or 1024 (INT4) of MMAs.
//
// A CTA walks a run of tiles: it waits for the MMAs of tile i, unpacks tile i + 1 into the one key buffer,
// issues its MMAs into the other half of the accumulator, and works on tile i's scores while they run. Two
// CTAs share an SM (one of twice the threads at head_dim 256; one where INT4 keys and FP32 queries, in two
// terms each, fill its shared memory). Codes are loaded a tile ahead into registers.
//
// 65536 tokens x 8 heads x 128 INT2, 32 queries x 4 query heads, both passes: 91 us, of which 30 are
// exponentials; a CTA's run of 14 tiles takes 83 thousand clocks (log-sum-exps) and 105 thousand (weights)
// from a cold cache, 5900 and 7500 a tile with the start: unpacking and the barriers' turns beside the
// exponentials. INT4: 118 us. FP32 queries: INT2 103 us, INT4 168 us.
#pragma once

#include "tma.cuh"
#include "weights_tc.cuh"

namespace kvb {
namespace weights_umma {

using weights_tc::as_log2;
using weights_tc::kLn2;
using weights_tc::kLog2e;
using weights_tc::kLowest;

constexpr int kTile = 128;              // places, and query rows, of a tile
constexpr int kBlockBytes = kTile * 128;  // 128 rows of 64 FP16: one swizzled block
constexpr uint32_t kColumns = 256;      // TMEM: two accumulators of 128 columns
constexpr int kMostSlots = 512;         // selected blocks that a CTA's run of places may touch

struct Job {
  WeightsArgs a;
  int rows;            // query rows a KV head
  int row0;            // the first of this launch's: CTAs (., ., z) take kTile from row0 + z kTile on
  int total_tiles, tiles_per_cta;
  int parts;           // parts per row in scratch (0: log-sum-exps given)
  int add;             // add to what out holds
};

// ---- tcgen05 (PTX ISA)

__device__ __forceinline__ void tmem_alloc(uint32_t where) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "r"(kColumns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns));
}
__device__ __forceinline__ void fence_before_sync() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after_sync() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_async_proxy() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Waits for a phase of the MMAs' barrier, a second at most. The clock is read only when the phase is not
// near: a read takes about as long as a tile's MMAs.
__device__ __forceinline__ bool wait_done(uint32_t bar, uint32_t parity) {
  for (int i = 0; i < 64; ++i)
    if (mbar_try(bar, parity)) return true;
  return mbar_wait_until(bar, parity, global_ns() + 1000000000ull, 1u << 26);
}

// Shared-memory matrix descriptor: K-major rows of 128 bytes with the 128-byte swizzle, groups of 8 rows
// 1024 bytes apart.
__device__ __forceinline__ uint64_t matrix(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// D[128 lanes, n columns] (+)= A B^T, FP16 operands, FP32 sums, 16 of K.
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, int n, bool add) {
  const uint32_t instruction = (1u << 4) | (static_cast<uint32_t>(n) >> 3 << 17) | (kTile >> 4 << 24);
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(instruction), "r"(static_cast<uint32_t>(add))
      : "memory");
}
// Arrives on `bar` when the MMAs issued so far are done.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// 32 columns of this warp's 32 lanes; the values are there after tmem_wait.
__device__ __forceinline__ void tmem_load32(uint32_t tmem, float (&v)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(tmem));
}
// Waits for the loads so far. It takes their values through, so that nothing uses them before.
__device__ __forceinline__ void tmem_wait(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(v[i]));
}

// Address of 16-byte chunk `chunk` (of 8) of row `row` of a swizzled block.
__device__ __forceinline__ uint32_t chunk_at(uint32_t block, int row, int chunk) {
  return block + row * 128 + ((chunk ^ (row & 7)) << 4);
}
__device__ __forceinline__ void store_chunk(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Threads of a place, or query row: warps w, w + 4, ... share the accumulator lanes of quarter w. Four where
// one CTA has the SM (head_dim 256, 252 rows x 23561 places INT2: 51.0 us, two 71.5); with two CTAs an SM
// two are faster (head_dim 128, 128 rows x 65536 places x 8 heads INT2: 86 us, four 103).
constexpr int shares(int d) { return d <= 128 ? 2 : 4; }
constexpr int threads(int d) { return 128 * shares(d); }
constexpr int resident(int d) { return d <= 128 ? 2 : 1; }  // CTAs on an SM

template <int BITS, int D, bool LO, bool LSE>
__global__ void __launch_bounds__(threads(D), resident(D)) weights_umma_kernel(const Job j, Divisor bt_by) {
  constexpr int kThreads = threads(D), kShares = shares(D), kChunks = 4 / kShares;  // 32-column chunks a share
  constexpr int kBlocks = (D + 63) / 64;        // swizzled blocks of a tile's row of FP16
  constexpr int kKeyTerms = BITS == 4 ? 2 : 1, kQueryTerms = LO ? 2 : 1;
  constexpr int kPieces = D / 32;               // 32-dim pieces of a row
  constexpr int kOwn = (kPieces + kShares - 1) / kShares;  // of them, a thread's
  constexpr int kWords = BITS;                  // 32-bit words of codes of a piece
  // all shares have whole pairs of pieces: they start on 16 bytes of INT2 codes, 4 of scales
  constexpr bool kEven = kPieces % (2 * kShares) == 0;
  extern __shared__ uint8_t raw_smem[];
  __shared__ uint64_t done_bar;
  __shared__ uint32_t tmem_at;
  __shared__ int gave_up;
  __shared__ alignas(16) float4 infos[kTile / 2];  // of two rows: factors, negated log-sum-exps
  __shared__ alignas(16) int seen[kTile];
  __shared__ float sums_of[2][kShares - 1][kTile];
  __shared__ float2 state[kShares - 1][kTile];
  __shared__ int2 slots[kMostSlots];  // (pool block, valid rows) of the run's selected blocks
  __shared__ uint32_t valid_mask[4][4];  // of tile i: [i & 3] (a warp may be a tile behind another)
  const WeightsArgs& a = j.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quarter = warp & 3, share = warp >> 2;
  const int row = quarter * 32 + lane;          // the place this thread unpacks; its accumulator lane
  const int h = blockIdx.y, gqa = a.qh / a.kvh, groups = D / a.group;
  const uint32_t base = (smem_addr(raw_smem) + 1023u) & ~1023u;
  const uint32_t keys = base, queries = base + kKeyTerms * kBlocks * kBlockBytes;
  const int places = a.n_sel * a.bt;
  const int first_tile = blockIdx.x * j.tiles_per_cta;
  const int tiles = min(j.total_tiles - first_tile, j.tiles_per_cta);
  const int row0 = j.row0 + blockIdx.z * kTile;
  const int rows = min(kTile, j.rows - row0);               // query rows of this CTA
  const int columns = LSE ? kTile : (rows + 31) / 32 * 32;  // of the accumulator

  if (threadIdx.x == 0) {
    gave_up = 0;
    mbar_init(smem_addr(&done_bar), 1);
    mbar_init_fence();
  }
  pdl_wait();
  // Behind the wait: a CTA launched early must not hold tensor memory that the grid it waits for needs.
  if (warp == 0) tmem_alloc(smem_addr(&tmem_at));
  pdl_launch();

  // ---- codes and scales of this thread's place, a tile ahead
  const int first_slot = divide(first_tile * kTile, bt_by);
  uint32_t code[kOwn][kWords];
  // Scales: in pairs, of two pieces each (groups of 32, kEven); of a piece's
  // two halves of 16 dims (groups of 16 or 48); or one a piece.
  uint32_t scale[kOwn];
  const bool in_pairs = a.group == 32 && kEven, in_halves = a.group % 32 != 0;
  bool valid = false;
  float prev = 0.f;
  const auto load = [&](int i) {
    valid = false;
    if (i >= tiles) return;
    const int place = (first_tile + i) * kTile + row;
    if (place >= places) return;
    const int slot = divide(place, bt_by), in_block = place - slot * a.bt;
    const int2 info = slots[slot - first_slot];
    const int blk = info.x;
    valid = in_block < info.y;
    if (!LSE && share == 0 && (a.previous || j.add))
      prev = j.add ? a.out[h * a.out_stride + place] : a.previous[h * a.previous_stride + place];
    if (!valid) return;
    const long long r = (static_cast<long long>(blk) * a.bt + in_block) * a.kvh + h;
    const uint8_t* from = a.kp + r * (D * BITS / 8);
    const __half* s = a.ks + r * groups;
    if constexpr (BITS == 2 && kEven) {  // two pieces in one access
#pragma unroll
      for (int k = 0; k < kOwn; k += 2) {
        const uint4 v = *reinterpret_cast<const uint4*>(from + (share * kOwn + k) * 8);
        code[k][0] = v.x, code[k][1] = v.y, code[k + 1][0] = v.z, code[k + 1][1] = v.w;
      }
    } else {
#pragma unroll
      for (int k = 0; k < kOwn; ++k) {
        const int piece = share * kOwn + k;
        if (piece >= kPieces) continue;
        if constexpr (BITS == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(from + piece * 16);
          code[k][0] = v.x, code[k][1] = v.y, code[k][2] = v.z, code[k][3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(from + piece * 8);
          code[k][0] = v.x, code[k][1] = v.y;
        }
      }
    }
    const unsigned short* u = reinterpret_cast<const unsigned short*>(s);
    if (in_pairs) {
#pragma unroll
      for (int k = 0; k < kOwn; k += 2) scale[k] = *reinterpret_cast<const uint32_t*>(u + share * kOwn + k);
    } else {
#pragma unroll
      for (int k = 0; k < kOwn; ++k) {
        const int piece = min(share * kOwn + k, kPieces - 1);
        if (a.group == 16) scale[k] = reinterpret_cast<const uint32_t*>(u)[piece];
        else if (in_halves) scale[k] = u[32 * piece / a.group] | static_cast<uint32_t>(u[(32 * piece + 16) / a.group]) << 16;
        else scale[k] = u[32 * piece / a.group];
      }
    }
  };
  // Dequantizes the loaded codes into the key blocks, `down` = 2^-4 where a scale is too large. Returns
  // whether one is.
  const auto unpack = [&](__half2 down) {
    bool large = false;
    if (!valid) return large;
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const int piece = share * kOwn + k;
      if (piece >= kPieces) continue;
      constexpr uint32_t kLimit = BITS == 4 ? 0x6FFFu : 0x77FFu;
      const uint32_t one = in_pairs ? scale[k & ~1] >> (16 * (k & 1)) & 0xFFFFu : scale[k];
      const uint32_t bits = in_halves ? one : one * 0x10001u;
      large |= (bits & 0x7FFFu) > kLimit || (bits >> 16 & 0x7FFFu) > kLimit;
      const __half2 two = __hmul2(u32_as_h2(bits), down);
      const __half2 s0 = __low2half2(two), s1 = __high2half2(two);
      const uint32_t block = keys + (piece >> 1) * kBlockBytes;
#pragma unroll
      for (int w = 0; w < 4; ++w) {  // 8 dims
        __half2 o[4];
        if constexpr (BITS == 4) {
          LanePairs<4>::centred(code[k][w], o);
        } else {
          __half2 all[8];
          LanePairs<2>::centred(code[k][w >> 1], all);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = all[4 * (w & 1) + i];
        }
        const __half2 s = w < 2 ? s0 : s1;
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __half2 v = __hmul2(o[i], s);
          hi[i] = h2_as_u32(v);
          if constexpr (BITS == 4) lo[i] = h2_as_u32(__hfma2(o[i], s, __hneg2(v)));
        }
        const uint32_t at = chunk_at(block, row, (piece & 1) * 4 + w);
        store_chunk(at, hi[0], hi[1], hi[2], hi[3]);
        if constexpr (BITS == 4) store_chunk(at + kBlocks * kBlockBytes, lo[0], lo[1], lo[2], lo[3]);
      }
    }
    return large;
  };
  const __half2 kOne = __float2half2_rn(1.f), kDown = __float2half2_rn(0.0625f);
  {
    const int last_slot = divide(min((first_tile + tiles) * kTile, places) - 1, bt_by);
    for (int i = threadIdx.x; i <= last_slot - first_slot; i += kThreads) {
      const int blk = a.table ? a.table[first_slot + i] : first_slot + i;
      int count = 0;
      if (blk < 0 || blk >= a.n_pool) {
        if (a.status) atomicOr(a.status, kDevBadBlockIndex);
      } else {
        count = a.valid[blk];
        if ((count < 0 || count > a.bt) && a.status) atomicOr(a.status, kDevBadValidCount);
      }
      slots[i] = make_int2(blk, count);
    }
    __syncthreads();
  }
  load(0);

  // ---- the query rows: kShares threads a row, taking turns at its units of 16 dims; their infos
  {
    constexpr int kUnits = D / 16, kMine = (kUnits + kShares - 1) / kShares;
    const int r = threadIdx.x / kShares, side = threadIdx.x % kShares, at = row0 + r;
    const bool live = r < rows;
    const int t = live ? at / gqa : 0, head = h * gqa + (live ? at % gqa : 0);
    const long long q = (static_cast<long long>(t) * a.qh + head) * D;
    int n = !live ? 0 : a.visible ? a.visible[t] : 0x7fffffff;
    const float given = a.lse_in && live ? a.lse_in[static_cast<long long>(t) * a.qh + head] : 0.f;
    float x[kMine][2][8] = {};
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int unit = side + kShares * k;
      if (!live || unit >= kUnits) continue;
      load_query8(a.query, a.dtype, q + 16 * unit, x[k][0]);
      load_query8(a.query, a.dtype, q + 16 * unit + 8, x[k][1]);
    }
    // a row that adds nothing may hold anything (padding): it enters the products as zeros, and sees nothing
    const bool enters = n > 0 && given != -INFINITY;
    if (!enters) n = 0;
#pragma unroll
    for (int k = 0; k < kMine; ++k)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (!enters) x[k][i >> 3][i & 7] = 0.f;
        top = fmaxf(top, fabsf(x[k][i >> 3][i & 7]));
      }
#pragma unroll
    for (int o = 1; o < kShares; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    int e = 0;
    if (top > 0.f && top < INFINITY) e = 14 - ilogbf(top);
    const auto power = [](int i) { return __int_as_float((i + 127) << 23); };
    const int e1 = e / 2, e2 = e - e1;
    // a negative scale goes into the query, so that the factor is not negative
    const float s1 = power(e1) * (a.sm_scale < 0.f ? -1.f : 1.f), s2 = power(e2);
    const float factor = fabsf(a.sm_scale) * kLog2e * power(-e1) * power(-e2);
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int unit = side + kShares * k;
      if (unit >= kUnits) continue;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // the order of the unpacked codes: two words of 8, or the halves of one word of 16
          const int d0 = BITS == 4 ? 8 * w + i : 4 * w + i, d1 = BITS == 4 ? d0 + 4 : d0 + 8;
          const float u = x[k][d0 >> 3][d0 & 7] * s1 * s2, v = x[k][d1 >> 3][d1 & 7] * s1 * s2;
          const __half hu = __float2half_rn(u), hv = __float2half_rn(v);
          hi[i] = h2_as_u32(__halves2half2(hu, hv));
          if constexpr (LO) lo[i] = h2_as_u32(__floats2half2_rn(u - __half2float(hu), v - __half2float(hv)));
        }
        const uint32_t to = chunk_at(queries + (unit >> 2) * kBlockBytes, r, (unit & 3) * 2 + w);
        store_chunk(to, hi[0], hi[1], hi[2], hi[3]);
        if constexpr (LO) store_chunk(to + kBlocks * kBlockBytes, lo[0], lo[1], lo[2], lo[3]);
      }
    }
    float l2 = LSE ? 0.f : INFINITY;
    if constexpr (!LSE) {
      const long long to = static_cast<long long>(t) * a.qh + head;
      if (j.parts) {  // (m, l) parts of the log-sum-exp, m in log2 units; all lanes take part
        const float2* part = reinterpret_cast<const float2*>(a.scratch) +
                             (static_cast<long long>(h) * j.rows + (live ? at : 0)) * j.parts;
        float m = kLowest, l = 0.f;
#pragma unroll 8
        for (int p = 0; p < j.parts; p += kShares) {
          const float2 v = p + side < j.parts ? part[p + side] : make_float2(kLowest, 0.f);
          const float up = fmaxf(m, v.x);
          l = l * fast_exp2(m - up) + v.y * fast_exp2(v.x - up);
          m = up;
        }
#pragma unroll
        for (int o = 1; o < kShares; o <<= 1) {
          const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l3 = __shfl_xor_sync(0xffffffffu, l, o);
          const float up = fmaxf(m, m2);
          l = l * fast_exp2(m - up) + l3 * fast_exp2(m2 - up);
          m = up;
        }
        l2 = l == 0.f ? -INFINITY : m + log2f(l);
        if (live && blockIdx.x == 0 && side == 0) a.lse[to] = l2 * kLn2;
        if (l2 == -INFINITY) l2 = INFINITY;
      } else if (live) {
        l2 = as_log2(given);
      }
      if (n <= 0) l2 = INFINITY;
    }
    if (side == 0) {
      float* pair = reinterpret_cast<float*>(infos + r / 2) + (r & 1);
      pair[0] = factor;
      pair[2] = -l2;
      seen[r] = n;
    }
  }

  // ---- tile 0
  const uint32_t bar = smem_addr(&done_bar);
  const auto issue = [&](int i) {  // one thread
    const uint32_t d = tmem_at + (i & 1) * kTile;
    bool add = false;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const uint32_t at = (k >> 2) * kBlockBytes + (k & 3) * 32;
#pragma unroll
      for (int term = 0; term < kKeyTerms + kQueryTerms - 1; ++term) {  // hi hi, lo hi, hi lo
        const bool key_lo = kKeyTerms == 2 && term == 1, query_lo = term == kKeyTerms;
        const uint64_t key = matrix(keys + (key_lo ? kBlocks * kBlockBytes : 0) + at);
        const uint64_t query = matrix(queries + (query_lo ? kBlocks * kBlockBytes : 0) + at);
        mma_f16(d, LSE ? query : key, LSE ? key : query, columns, add);
        add = true;
      }
    }
    mma_commit(bar);
  };
  // Unpacks the loaded tile i, makes it visible to the MMAs, and issues them. All threads; the barrier in
  // the middle also ends the work on the accumulator that they overwrite. `large`: the tile's scores have
  // to be multiplied by 16. `stop`: some thread's wait has run out (`timed_out`); the second barrier of
  // the rare path keeps the flag as it is until all have read it.
  bool mine_valid = false, stop = false;
  float mine_prev = 0.f;
  const auto advance = [&](int i, bool timed_out) {
    bool large = false;
    mine_valid = valid;
    if (timed_out) gave_up = 1;
    if (i < tiles) {
      large = unpack(kOne);
      mine_prev = prev;
      const uint32_t mask = __ballot_sync(0xffffffffu, valid);
      if (share == 0 && lane == 0) valid_mask[i & 3][quarter] = mask;
    }
    fence_async_proxy();
    fence_before_sync();
    large = __syncthreads_or(large || timed_out);
    fence_after_sync();
    if (large) {
      stop = gave_up;
      unpack(kDown);
      fence_async_proxy();
      __syncthreads();
    }
    if (i < tiles && threadIdx.x == 0 && !stop) issue(i);
    return large;
  };
  bool next_large = advance(0, false);
  bool next_valid = mine_valid;
  float next_prev = mine_prev;
  load(1);
  int all_see = 0x7fffffff;  // places below are seen by every row that sees anything
  bool any = false;
  for (int i = lane; i < rows; i += 32)
    if (seen[i] > 0) all_see = min(all_see, seen[i]), any = true;
  all_see = __reduce_min_sync(0xffffffffu, all_see);
  if (!__any_sync(0xffffffffu, any)) all_see = 0;

  const float own_factor = reinterpret_cast<const float*>(infos + row / 2)[row & 1];
  const int own_seen = seen[row];
  const uint32_t lanes_at = static_cast<uint32_t>(quarter * 32) << 16;
  float run_m = kLowest, run_l = 0.f;  // LSE: of query row `row` over this share of the columns
  float sum = 0.f, sum_prev = 0.f;     // weights: of the last tile's place `row`, this share

  const auto write = [&](int i) {
    const int place = (first_tile + i) * kTile + row;
    if (place >= places) return;
    float all = sum;
#pragma unroll
    for (int k = 0; k < kShares - 1; ++k) all += sums_of[i & 1][k][row];
    a.out[h * a.out_stride + place] = sum_prev + all;
  };

  int i = 0;
  for (; i < tiles; ++i) {
    const bool timed_out = !wait_done(bar, i & 1);
    fence_after_sync();
    const bool large = next_large, place_valid = next_valid;
    const float place_prev = next_prev;
    next_large = advance(i + 1, timed_out);
    next_valid = mine_valid;
    next_prev = mine_prev;
    if (stop) break;  // all threads
    if (!LSE && share == 0 && i > 0) write(i - 1);  // the other shares' sums have arrived
    load(i + 2);

    const int place0 = (first_tile + i) * kTile;
    const uint32_t acc = tmem_at + (i & 1) * kTile + lanes_at;
    if constexpr (LSE) {
      const uint32_t* mask = valid_mask[i & 3] + kChunks * share;
      bool full = place0 + kTile <= all_see;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) full = full && mask[c] == 0xFFFFFFFFu;
      const float scaled = large ? own_factor * 16.f : own_factor;
      const int column0 = share * 32 * kChunks;
      float chunks[kChunks][32];
      tmem_load32(acc + column0, chunks[0]);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        float (&v)[32] = chunks[c];
        tmem_wait(v);
        if (c + 1 < kChunks) tmem_load32(acc + column0 + 32 * (c + 1), chunks[(c + 1) % kChunks]);  // while these are worked on
        if (!full) {
          const int see = own_seen - (place0 + column0 + c * 32);  // columns seen
          const uint32_t live = mask[c] & (see <= 0 ? 0u : see >= 32 ? 0xFFFFFFFFu : (1u << see) - 1u);
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] = live >> k & 1u ? v[k] * scaled : -INFINITY;
        }
        const float factor = full ? scaled : 1.f;
        float tops[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int k = 4; k < 32; ++k) tops[k & 3] = fmaxf(tops[k & 3], v[k]);
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * factor;
        if (top > run_m + 8.f) {  // the running max moves only past 2^8: terms stay finite
          run_l *= fast_exp2(run_m - top);
          run_m = top;
        }
        F2 part[2] = {f2(0.f), f2(0.f)};
        const F2 by = f2(factor), less = f2(-run_m);
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const float2 x = parts(fma2(f2(v[k], v[k + 1]), by, less));
          part[k / 2 & 1] = add2(part[k / 2 & 1], f2(fast_exp2(x.x), fast_exp2(x.y)));
        }
        const float2 sums = parts(add2(part[0], part[1]));
        run_l += sums.x + sums.y;
      }
    } else {
      const bool full = place0 + kTile <= all_see;
      F2 part[2] = {f2(0.f), f2(0.f)};
      // the columns' chunks of 32 alternate between the shares
      float chunks[kChunks][32];
      if (share * 32 < columns) tmem_load32(acc + share * 32, chunks[0]);
#pragma unroll
      for (int n = 0; n < kChunks; ++n) {
        const int c = (share + n * kShares) * 32, next = c + kShares * 32;
        if (c >= columns) break;
        float (&v)[32] = chunks[n];
        tmem_wait(v);
        if (n + 1 < kChunks && next < columns) tmem_load32(acc + next, chunks[(n + 1) % kChunks]);  // while these are worked on
        if (large) {
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] *= 16.f;
        }
        const float4* info = infos + c / 2;
        const int place = place0 + row;
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const float4 two = info[k / 2];
          float2 x = parts(fma2(f2(v[k], v[k + 1]), f2(two.x, two.y), f2(two.z, two.w)));
          if (!full) {
            if (place >= seen[c + k]) x.x = -INFINITY;
            if (place >= seen[c + k + 1]) x.y = -INFINITY;
          }
          part[k / 2 & 1] = add2(part[k / 2 & 1], f2(fast_exp2(x.x), fast_exp2(x.y)));
        }
      }
      const float2 sums = parts(add2(part[0], part[1]));
      sum = place_valid ? sums.x + sums.y : 0.f;
      sum_prev = place_prev;
      if (share > 0) sums_of[i & 1][share - 1][row] = sum;
    }
  }

  if (stop) {  // the MMAs' barrier did not complete in a second: nothing plausible is left behind
    if (threadIdx.x == 0 && a.status) atomicOr(a.status, kDevStreamTimeout);
    wait_done(bar, i & 1);
    const float nan = __int_as_float(0x7fffffff);
    run_l = run_m = nan;
    if (!LSE && share == 0)
      for (int t = max(i - 1, 0); t < tiles; ++t) {
        const int place = (first_tile + t) * kTile + row;
        if (place < places) a.out[h * a.out_stride + place] = nan;
      }
  }
  fence_before_sync();
  __syncthreads();
  if constexpr (LSE) {
    if (share > 0) state[share - 1][row] = make_float2(run_m, run_l);
    __syncthreads();
    if (share == 0 && row < rows) {
      float2 part = make_float2(run_m, run_l);
#pragma unroll
      for (int k = 0; k < kShares - 1; ++k) {
        const float2 other = state[k][row];
        const float top = fmaxf(part.x, other.x);
        part = make_float2(top, part.y * fast_exp2(part.x - top) + other.y * fast_exp2(other.x - top));
      }
      if (own_seen <= 0) part = make_float2(kLowest, 0.f);
      if (stop) part = make_float2(0.f, __int_as_float(0x7fffffff));
      reinterpret_cast<float2*>(a.scratch)[(static_cast<long long>(h) * j.rows + row0 + row) * j.parts +
                                           blockIdx.x] = part;
    }
  } else if (share == 0 && !stop) {
    write(tiles - 1);
  }
  if (warp == 0) tmem_free(tmem_at);
}

// Query rows from which the 128-row tiles pay; keys and queries in two terms each are too large for the
// shared memory at head_dim 256.
template <int BITS, int D, bool LO>
bool takes(const WeightsArgs& a) {
  return a.queries * (a.qh / a.kvh) > 32 && !(D == 256 && BITS == 4 && LO);
}

template <int BITS, int D, bool LO, bool LSE>
cudaError_t launch_pass(Job j, cudaStream_t s) {
  constexpr int kBlocks = (D + 63) / 64;
  constexpr int smem = ((BITS == 4 ? 2 : 1) + (LO ? 2 : 1)) * kBlocks * kBlockBytes + 1024;
  const auto kernel = weights_umma_kernel<BITS, D, LO, LSE>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const int ctas = (j.total_tiles + j.tiles_per_cta - 1) / j.tiles_per_cta;
  const int chunks = (j.rows + kTile - 1) / kTile;
  // log-sum-exps of different rows are independent; the weights of later rows add to those before
  const int z = LSE && chunks <= 65535 ? chunks : 1;
  for (j.row0 = 0; j.row0 < j.rows; j.row0 += z * kTile) {
    j.add = j.row0 > 0;
    const cudaError_t l = launch_pdl(kernel, dim3(ctas, j.a.kvh, z), threads(D), smem, s, j,
                                     divisor(static_cast<unsigned>(j.a.bt)));
    if (l != cudaSuccess) return l;
  }
  return cudaSuccess;
}

struct Plan {
  int total_tiles, tiles_per_cta, parts;
};
inline Plan plan(int n_sel, int bt, int kvh, int ctas) {  // ctas: on an SM
  Plan p;
  p.total_tiles = static_cast<int>((static_cast<long long>(n_sel) * bt + kTile - 1) / kTile);
  const int want = 148 * ctas / kvh < 1 ? 1 : 148 * ctas / kvh;
  p.tiles_per_cta = (p.total_tiles + want - 1) / want;
  // a run touches at most this many blocks (a partial one at either end): more CTAs otherwise
  const long long most = static_cast<long long>(kMostSlots - 2) * bt / kTile;
  if (p.tiles_per_cta > most) p.tiles_per_cta = most < 1 ? 1 : static_cast<int>(most);
  p.parts = (p.total_tiles + p.tiles_per_cta - 1) / p.tiles_per_cta;
  return p;
}

template <int BITS, int D, bool LO>
cudaError_t launch(const WeightsArgs& a, cudaStream_t s) {
  Job j{};
  j.a = a;
  j.rows = a.queries * (a.qh / a.kvh);
  const Plan p = plan(a.n_sel, a.bt, a.kvh, resident(D));
  j.total_tiles = p.total_tiles;
  j.tiles_per_cta = p.tiles_per_cta;
  if (!a.lse_in) {
    j.parts = p.parts;
    if (j.parts > a.parts_room) return cudaErrorInvalidValue;
    const cudaError_t e = launch_pass<BITS, D, LO, true>(j, s);
    if (e != cudaSuccess) return e;
  }
  return launch_pass<BITS, D, LO, false>(j, s);
}

}  // namespace weights_umma
}  // namespace kvb
