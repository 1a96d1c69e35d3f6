// Attention of the newest tokens of a batch over a paged cache (single tokens, or a few drafted ones), with the keys that
// a group of sequences shares read once for all of them.
//
// A call is a chain of launches: plan (who reads what; not for few rows), prefix units (only with groups: attn_prefix.cu), own units, join.
// Each comes up while the one before still runs and waits for its end before it reads anything: what the plan wrote two launches ago
// is visible behind that wait only.  (Own units that began beside the prefix units, and a join that read the plan early, took 2 to 4 us less
// of a call with groups, 1 us of one without, on an order that nothing promised.)  For 32 sequences of 600 keys behind 8219 shared
// ones (32 query and 8 kv heads, D 128, bf16) that is 34.6 us in a graph: plan 5, prefix 13.5, own units and join 16, against 11 us for the bytes; what is
// left is the latency of the chain.  One sequence of 1000 keys (f16, D 64) takes 9.6 us.
//
// Own units are bound by memory: a key and a value are used by the few query rows of one sequence, so the kernel is a
// stream of pages through shared memory, with tiles asked for by TMA several tiles ahead: 32 sequences of up to 8k keys, 537
// MB of bf16, take 98 us with all launches (5.5 TB/s), 268 MB of E4M3 60 us.  Scores and values go through mma.sync m16n8k16:
// with 4 to 16 query rows a tcgen05 tile of 128 rows would be empty for the most part, and up to 16 rows the products of a tile
// take less time than its bytes.  With 64 rows they do not any more (bf16 237 us).
#include "attn_paged.cuh"

#include <cmath>
#include <cstddef>
#include <type_traits>

namespace fa4b {

// ---- plan -------------------------------------------------------------------------------------------------------------
// One CTA, and every other launch of the call waits for it.  More warps would walk the same instructions and cost more than
// they help (1024 threads took 7.1 us for 32 sequences, these 5), and what is sums over items a warp does alone: three of them at once
// for the three lines of sums, without a barrier.
constexpr int kPlanThreads = 256;

__device__ __noinline__ uint32_t paged_div(uint32_t a, uint32_t b) { return a / b; }

// Exclusive prefix sums of a[0..n) in shared memory, in place, by one warp; returns the total.
__device__ __noinline__ int warp_scan(int* a, int n) {
  const int lane = threadIdx.x & 31;
  int total = 0;
#pragma unroll 1
  for (int base = 0; base < n; base += 32) {
    const int i = base + lane, v = i < n ? a[i] : 0;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (i < n) a[i] = total + x - v;
    total += __shfl_sync(0xffffffffu, x, 31);
  }
  return total;
}

// How a line is cut, by one warp.  Items i < n have units[i] (or `each`) units of tiles[i] tiles.  A piece that ends one unit
// and begins another pays for the beginning of both (about `extra` tiles), so pieces that keep to one unit are best where they are no
// longer for it: the shortest such length for which the pieces of all units are no more than the workers.  Otherwise the line
// with `extra` tiles put before each unit is cut at equal distances.
__device__ __noinline__ PagedCut warp_cut(const int* tiles, const int* units, int n, uint32_t each, uint32_t workers, uint32_t extra, uint32_t least) {
  const int lane = threadIdx.x & 31;
  uint32_t all = 0u, all_units = 0u;
#pragma unroll 1
  for (int i = lane; i < n; i += 32) {
    const uint32_t u = tiles[i] ? (units ? (uint32_t)units[i] : each) : 0u;
    all += u * tiles[i], all_units += u;
  }
  all = __reduce_add_sync(0xffffffffu, all), all_units = __reduce_add_sync(0xffffffffu, all_units);
  const uint32_t line = max(paged_div(all + all_units * extra + workers - 1, workers), least + extra);
  uint32_t per = max(paged_div(all + workers - 1, workers), least);
  if (all_units <= workers)
#pragma unroll 1
    for (int tries = 0; tries < 8 && per <= line; ++tries, ++per) {
      uint32_t pieces = 0u;
#pragma unroll 1
      for (int i = lane; i < n; i += 32) pieces += (units ? (uint32_t)units[i] : each) * paged_div(tiles[i] + per - 1, per);
      if (__reduce_add_sync(0xffffffffu, pieces) <= workers) return {per, 0u, 1u};
    }
  return {line, extra, 0u};
}

// The last i in [0, n) with cum[i] <= x.
__device__ __noinline__ int paged_find(const int* cum, int n, uint32_t x) {
  int lo = 0, hi = n - 1;
#pragma unroll 1
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((uint32_t)cum[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// dynamic shared memory of the plan, in words
__host__ __device__ inline size_t paged_plan_words(int n, int groups) { return 4 * (size_t)n + 6 * (size_t)groups + 1; }

// Lengths, groups, and the lines of tiles.  The shared part of a group is what the caller says, cut to what every query row
// of every member sees (so that no row of a prefix unit needs a mask) and to whole 16 keys; a group of one member has none.
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PagedParams p) {
  __shared__ int bad;
  __shared__ PagedLine s_own, s_prefix;
  extern __shared__ int dyn[];
  int* own_cum = dyn;                  // [n]
  int* s_slot = own_cum + p.n;         // [n]
  int* s_len = s_slot + p.n;           // [n]
  int* s_group = s_len + p.n;          // [n] -1: none
  int* offsets = s_group + p.n;        // [groups + 1]
  int* g_shared = offsets + p.groups + 1;  // [groups] shortest member's length - T, then the shared keys
  int* g_first = g_shared + p.groups;  // [groups] a member with keys
  int* g_count = g_first + p.groups;   // [groups] members with keys, then whether a shared page is missing
  int* g_cum = g_count + p.groups;     // [groups]
  int* g_unit = g_cum + p.groups;      // [groups]
  constexpr int nt = kPlanThreads;
  const int tid = threadIdx.x, warp = tid >> 5;
  pdl_trigger();
  if (tid == 0) bad = 0;
#pragma unroll 1
  for (int g = tid; g < p.groups; g += nt) g_shared[g] = INT_MAX, g_first[g] = INT_MAX, g_count[g] = 0;
  pdl_wait();
#pragma unroll 1
  for (int g = tid; g <= p.groups && p.groups > 0; g += nt) offsets[g] = p.offsets[g];
#pragma unroll 1
  for (int i = tid; i < p.n; i += nt) {
    const int slot = p.seqs ? p.seqs[i] : i;
    s_slot[i] = slot, s_group[i] = p.groups > 0 ? -1 : 0;
    s_len[i] = (uint32_t)slot < (uint32_t)p.c.max_seqs ? min(max(p.c.lens[slot], 0), p.c.width << p.c.page_shift) : 0;
  }
  __syncthreads();
  if (p.groups > 0) {
    // groups have to lie behind one another: the slots of their units are counted on it
#pragma unroll 1
    for (int g = tid; g < p.groups; g += nt)
      if (offsets[g] < 0 || offsets[g + 1] < offsets[g] || offsets[g + 1] > p.n) bad = 1;
#pragma unroll 1
    for (int i = tid; i < p.n; i += nt) {
      const int g = paged_find(offsets, p.groups, (uint32_t)i);  // the last group that begins at or before i
      if (i < offsets[g] || i >= offsets[g + 1]) continue;
      s_group[i] = g;
      if (s_len[i] > 0) {
        atomicMin(g_shared + g, max(s_len[i] - p.T, 0));
        atomicMin(g_first + g, i);
        atomicAdd(g_count + g, 1);
      }
    }
    __syncthreads();
    if (bad != 0) {
      if (tid == 0 && atomicCAS(p.status, 0u, 2u) == 0u) p.status[1] = (uint32_t)p.groups;
#pragma unroll 1
      for (int i = tid; i < p.n; i += nt) s_group[i] = -1;
    }
#pragma unroll 1
    for (int g = tid; g < p.groups; g += nt) {
      g_shared[g] = g_count[g] > 1 && bad == 0 ? min(max(p.shared[g], 0), g_shared[g]) & ~(kPagedAlign - 1) : 0;
      g_count[g] = 0;
    }
    __syncthreads();
    // A shared page that the table does not name: the group goes without, the own units know how to leave such a page out.
    const int shift = max(5, 8 - (31 - __clz(2 * p.groups - 1)));  // 2^shift threads for a group: a warp at least
#pragma unroll 1
    for (int g = tid >> shift; g < p.groups; g += nt >> shift) {
      const int pages = (g_shared[g] + p.c.page_tokens - 1) >> p.c.page_shift;
      const int32_t* row = p.c.table + (pages ? (int64_t)s_slot[g_first[g]] * p.c.table_stride : 0);
      bool missing = false;
#pragma unroll 1
      for (int j = tid & ((1 << shift) - 1); j < pages; j += 8 << shift) {
        int e[8];  // all on their way at once
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = j + (k << shift) < pages ? row[j + (k << shift)] : 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) missing |= (uint32_t)e[k] >= (uint32_t)p.c.pages;
      }
      if (missing) g_count[g] = 1;
    }
    __syncthreads();
#pragma unroll 1
    for (int g = tid; g < p.groups; g += nt) {
      const int shared = g_count[g] ? 0 : g_shared[g];
      const int units = shared ? p.c.heads * (((offsets[g + 1] - offsets[g]) * p.R + p.prefix_rows - 1) >> p.prefix_shift) : 0;
      g_shared[g] = shared;
      g_unit[g] = units;
      g_cum[g] = (shared + kPagedPrefixTile - 1) / kPagedPrefixTile;
    }
  }
#pragma unroll 1
  for (int i = tid; i < p.n; i += nt) {
    const int g = s_group[i];
    own_cum[i] = g < 0 ? 0 : own_tiles(p, p.groups > 0 && s_len[i] > 0 ? g_shared[g] : 0, s_len[i]);
  }
  __syncthreads();
  // warps 0, 1: the cuts and lines; warp 2: the numbers of units
  if (warp < 2) {
    const bool own = warp == 0;
    int* tiles = own ? own_cum : g_cum;
    const int* units = own ? nullptr : g_unit;
    const int n = own ? p.n : p.groups;
    const PagedCut cut = warp_cut(tiles, units, n, p.own_units, own ? p.own_workers : p.prefix_workers, own ? p.own_extra : p.prefix_extra, own ? p.own_min : 1);
#pragma unroll 1
    for (int i = tid & 31; i < n; i += 32) tiles[i] = (own ? 1 : units[i]) * (int)cut.length(tiles[i]);
    __syncwarp();
    const int total = warp_scan(tiles, n);
    if ((tid & 31) == 0) (own ? s_own : s_prefix) = {(uint32_t)total, cut};
  }
  __syncthreads();
  if (warp == 2) warp_scan(g_unit, p.groups);
  const int own_total = s_own.total;
  // the line of the own units has p.own_units of each entry of own_cum
  uint32_t line = (uint32_t)own_total * p.own_units;
  if ((uint64_t)own_total * p.own_units >= INT_MAX) {  // beyond what positions count: nothing is computed
    if (tid == 0 && atomicCAS(p.status, 0u, 3u) == 0u) p.status[1] = (uint32_t)own_total;
    line = 0u;
  }
  if (tid == 0) *p.head = {{line, s_own.cut}, s_prefix};
  __syncthreads();
  // all is known: the records
#pragma unroll 1
  for (int i = tid; i < p.n; i += nt) {
    const int g = max(s_group[i], 0), first = p.groups > 0 && s_len[i] > 0 ? g_shared[g] : 0;
    int4* r = reinterpret_cast<int4*>(p.seq + i);
    r[0] = make_int4(s_slot[i], s_len[i], first, own_cum[i]);
    p.own_cum[i] = own_cum[i];
    r[2] = make_int4(s_group[i] < 0 || line == 0u && own_total > 0, first > 0 ? (offsets[g + 1] - offsets[g]) * p.R : 0, 0, 0);
    if (first > 0) r[1] = make_int4(offsets[g], ((offsets[g + 1] - offsets[g]) * p.R + p.prefix_rows - 1) >> p.prefix_shift, g_unit[g], g_cum[g]);
  }
#pragma unroll 1
  for (int g = tid; g < p.groups; g += nt) {
    int4* r = reinterpret_cast<int4*>(p.group + g);
    const int shared = g_shared[g], rows = (offsets[g + 1] - offsets[g]) * p.R;
    r[0] = make_int4(shared, shared ? s_slot[g_first[g]] : 0, offsets[g], rows);
    p.g_cum[g] = g_cum[g];
    r[1] = make_int4(g_cum[g], g_unit[g], (rows + p.prefix_rows - 1) >> p.prefix_shift, 0);
  }
}

// The plan of a call of up to 32 rows without groups, a row to a lane: two rounds of loads and two sums, which a CTA of the own units
// works out sooner than a launch before it does; the first of them writes it down for the join.  `cum`: 32 words of shared memory of this warp's.
constexpr int kSmallRows = 32;
struct PagedSmall {
  int slot, len, cum, left_alone;  // of row `lane`
  PagedLine line;
};
__device__ __forceinline__ PagedSmall paged_small(const PagedParams& p, int* cum) {
  const int lane = threadIdx.x & 31;
  PagedSmall s;
  s.slot = lane < p.n ? (p.seqs ? p.seqs[lane] : lane) : -1;
  s.len = (uint32_t)s.slot < (uint32_t)p.c.max_seqs ? min(max(p.c.lens[s.slot], 0), p.c.width << p.c.page_shift) : 0;
  const int tiles = own_tiles(p, 0, s.len);
  cum[lane] = tiles;
  __syncwarp();
  const PagedCut cut = warp_cut(cum, nullptr, p.n, p.own_units, p.own_workers, p.own_extra, p.own_min);
  __syncwarp();
  cum[lane] = (int)cut.length(tiles);
  __syncwarp();
  const int total = warp_scan(cum, p.n);
  __syncwarp();
  s.cum = cum[lane];
  const bool fits = (uint64_t)total * p.own_units < INT_MAX;  // positions are counted in 32 bits
  s.line = {fits ? (uint32_t)total * p.own_units : 0u, cut};
  s.left_alone = !fits;
  if (!fits && blockIdx.x == 0 && lane == 0 && atomicCAS(p.status, 0u, 3u) == 0u) p.status[1] = (uint32_t)total;
  return s;
}

// ---- the units over keys of one sequence ------------------------------------------------------------------------------
// Sixteen query rows of a unit as one warp holds them: rows quad and quad + 8 of the fragments, accumulators over D, running
// maximum and sum.  Compute type: the cache's own 16-bit type, or f16 for an E4M3 cache (every E4M3 value is exact in f16;
// bf16 queries are brought into its range by a power of two per row, exact down to 2^-38 of the row's largest).
template <int D, bool kE4M3, typename QT>
struct PagedRows {
  using Mma = typename std::conditional<kE4M3, TagF16, QT>::type;
  static constexpr int kBoxBytes = D * (kE4M3 ? 1 : 2) < 128 ? D : 128;  // of a row, side by side in one box of shared memory
  uint32_t q[D / 16][4];
  float acc[D / 8][4], scale[2], m[2], l[2];
  int limit[2];  // the row sees keys below

  __device__ __forceinline__ void start(const PagedParams& p, const PagedUnit& u, int row0) {
    const int lane = threadIdx.x & 31, quad = lane >> 2, c4 = lane & 3;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = row0 + half * 8 + quad;
      const bool there = row < u.rows;
      const PagedRow r = paged_row(p, u, there ? row : 0);
      const uint8_t* src = p.q + 2 * (r.i * p.q_sb + r.h * p.q_sh + r.t * p.q_st);
      limit[half] = u.key_hi - (p.T - 1 - r.t);
      scale[half] = p.scale_log2 * (kE4M3 ? p.k_scale[u.head] : 1.f);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        if constexpr (kE4M3) {  // four neighbours: a thread's K codes are four neighbours too (see the scores below)
          const uint2 x = there ? *reinterpret_cast<const uint2*>(src + 2 * (k * 16 + c4 * 4)) : make_uint2(0u, 0u);
          q[k][half] = x.x, q[k][half + 2] = x.y;
        } else {
          q[k][half] = there ? *reinterpret_cast<const uint32_t*>(src + 2 * (k * 16 + c4 * 2)) : 0u;
          q[k][half + 2] = there ? *reinterpret_cast<const uint32_t*>(src + 2 * (k * 16 + 8 + c4 * 2)) : 0u;
        }
      }
      if constexpr (kE4M3 && std::is_same<QT, TagBf16>::value) {
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const float2 f = unpack16(q[k][half + e], TagBf16{});
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const RowShift to_f16 = row_shift(top);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int x = 0; x < 4; x += 2) {
            q[k][half + x] = bf16x2_shifted(q[k][half + x], to_f16);
          }
        scale[half] = scale[half] / to_f16.a / to_f16.b;
      }
      m[half] = -INFINITY, l[half] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < D / 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  }

  // kKeys keys from key0 on, at row `at` of a tile of kTileRows keys in shared memory; `valid`: a bit per 16 of them, the
  // table names a page of the pool
  template <int kKeys, int kTileRows>
  __device__ __forceinline__ void tile(const PagedUnit& u, const uint8_t* ktile, const uint8_t* vtile, int at, int key0, uint32_t valid) {
    const int lane = threadIdx.x & 31, c4 = lane & 3;
    const uint32_t kbase = smem_u32(ktile), vbase = smem_u32(vtile);
    constexpr uint32_t kAllValid = (1u << (kKeys / 16)) - 1u;
    // not every key of these is there for every row
    const bool special = key0 < u.key_lo || key0 + kKeys > u.key_all || (valid & kAllValid) != kAllValid;
    float sc[kKeys / 8][4];
#pragma unroll
    for (int j = 0; j < kKeys / 8; ++j) {
      sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
      const uint32_t row = at + j * 8 + (lane & 7);
      if constexpr (kE4M3) {
        // a matrix of ldmatrix is 8 keys x 16 codes, four neighbours to a thread: they stand in for k = 2c, 2c+1, 2c+8, 2c+9 of
        // the fragment, and the query fragments hold the same four neighbours there
#pragma unroll
        for (int x = 0; x < D / 64; ++x) {
          uint32_t b[4];
          ldmatrix4(b, kbase + swizzled_offset(row, x * 64 + (lane >> 3) * 16, kBoxBytes));
#pragma unroll
          for (int e = 0; e < 4; ++e) mma16816(sc[j], q[x * 4 + e], e4m3x2_to_f16x2(b[e]), e4m3x2_to_f16x2(b[e] >> 16), Mma{});
        }
      } else {
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
          uint32_t b[4];
          const uint32_t col = x * 64 + (lane >> 3) * 16;  // bytes of the row
          ldmatrix4(b, kbase + (col >> 7) * (kTileRows * 128) + swizzled_offset(row, col & 127u, 128));
          mma16816(sc[j], q[2 * x], b[0], b[1], Mma{});
          mma16816(sc[j], q[2 * x + 1], b[2], b[3], Mma{});
        }
      }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < kKeys / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = sc[j][e] * scale[e >> 1];
        if (special) {
          const int key = key0 + j * 8 + c4 * 2 + (e & 1);
          if (key < u.key_lo || key >= limit[e >> 1] || !(valid >> (j >> 1) & 1u)) x = -INFINITY;
        }
        sc[j][e] = x;
        top[e >> 1] = fmaxf(top[e >> 1], x);
      }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
    }
    // The reference point of a row moves only when its maximum has grown by more than 2^8 (probabilities then stay below
    // 2^8, which costs 16-bit ones no precision): most tiles leave the accumulators alone.
    if (__any_sync(0xffffffffu, top[0] > m[0] + 8.f || top[1] > m[1] + 8.f)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float next = fmaxf(m[h], top[h]);
        const float f = next == -INFINITY ? 1.f : paged_ex2(m[h] - next);
        m[h] = next;
        l[h] *= f;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) acc[j][2 * h] *= f, acc[j][2 * h + 1] *= f;
      }
    }
    const float m0 = m[0] == -INFINITY ? 0.f : m[0], m1 = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll
    for (int j = 0; j < kKeys / 8; ++j) {
      sc[j][0] = paged_ex2(sc[j][0] - m0), sc[j][1] = paged_ex2(sc[j][1] - m0);
      sc[j][2] = paged_ex2(sc[j][2] - m1), sc[j][3] = paged_ex2(sc[j][3] - m1);
      l[0] += sc[j][0] + sc[j][1], l[1] += sc[j][2] + sc[j][3];
    }
    // Values.  A key that is not there, or that some row must not see, has probability 0 for those rows, and 0 times what its
    // value may hold (anything, beyond the length) need not be 0: such keys are taken out of the product on both sides,
    // and those that some rows do see (the newest T - 1) are added row by row behind it.
#pragma unroll
    for (int kk = 0; kk < kKeys / 16; ++kk) {
      uint32_t a[4] = {pack16(sc[2 * kk][0], sc[2 * kk][1], Mma{}), pack16(sc[2 * kk][2], sc[2 * kk][3], Mma{}),
                       pack16(sc[2 * kk + 1][0], sc[2 * kk + 1][1], Mma{}), pack16(sc[2 * kk + 1][2], sc[2 * kk + 1][3], Mma{})};
      uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
      if (special) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = key0 + kk * 16 + h * 8 + c4 * 2;
          const bool ok = valid >> kk & 1u;
          keep[h] = (ok && key >= u.key_lo && key < u.key_all ? 0x0000ffffu : 0u) | (ok && key + 1 >= u.key_lo && key + 1 < u.key_all ? 0xffff0000u : 0u);
          a[2 * h] &= keep[h], a[2 * h + 1] &= keep[h];
        }
      }
      const uint32_t row = at + kk * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
      if constexpr (kE4M3) {
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {  // matrices: keys 0-7 and 8-15 of 16 codes, then of the next 16
          uint32_t b[4];
          ldmatrix4_trans(b, vbase + swizzled_offset(row, x * 32 + (lane >> 4) * 16, kBoxBytes));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // a register holds (key, key + 1) x (d, d + 1): even and odd d go to accumulators of their own
            uint32_t lo0 = e4m3x2_to_f16x2(__byte_perm(b[2 * e], 0, 0x4420)), lo1 = e4m3x2_to_f16x2(__byte_perm(b[2 * e + 1], 0, 0x4420));
            uint32_t hi0 = e4m3x2_to_f16x2(__byte_perm(b[2 * e], 0, 0x4431)), hi1 = e4m3x2_to_f16x2(__byte_perm(b[2 * e + 1], 0, 0x4431));
            if (special) lo0 &= keep[0], lo1 &= keep[1], hi0 &= keep[0], hi1 &= keep[1];
            mma16816(acc[4 * x + 2 * e], a, lo0, lo1, Mma{});
            mma16816(acc[4 * x + 2 * e + 1], a, hi0, hi1, Mma{});
          }
        }
      } else {
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
          uint32_t b[4];
          const uint32_t col = x * 32 + (lane >> 4) * 16;
          ldmatrix4_trans(b, vbase + (col >> 7) * (kTileRows * 128) + swizzled_offset(row, col & 127u, 128));
          if (special) b[0] &= keep[0], b[1] &= keep[1], b[2] &= keep[0], b[3] &= keep[1];
          mma16816(acc[2 * x], a, b[0], b[1], Mma{});
          mma16816(acc[2 * x + 1], a, b[2], b[3], Mma{});
        }
      }
    }
    if (key0 + kKeys > u.key_all) {
#pragma unroll 1
      for (int kk = max(0, u.key_all - key0); kk < min(kKeys, u.key_hi - key0); ++kk) {
        if (!(valid >> (kk >> 4) & 1u)) continue;
        const int from = (lane & ~3) | ((kk & 7) >> 1);
        float mine[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < kKeys / 8; ++j)
          if (j == kk >> 3) mine[0] = kk & 1 ? sc[j][1] : sc[j][0], mine[1] = kk & 1 ? sc[j][3] : sc[j][2];
        const float p0 = __shfl_sync(0xffffffffu, mine[0], from), p1 = __shfl_sync(0xffffffffu, mine[1], from);
        const bool see0 = key0 + kk < limit[0], see1 = key0 + kk < limit[1];
        const uint32_t row = at + kk;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          float2 f;
          if constexpr (kE4M3) {  // accumulators 2x and 2x + 1: d = 16 x + 4 c + {0, 2} and {1, 3}
            const uint32_t four = *reinterpret_cast<const uint32_t*>(vtile + swizzled_offset(row, (j >> 1) * 16 + c4 * 4, kBoxBytes));
            f = unpack16(e4m3x2_to_f16x2(__byte_perm(four, 0, j & 1 ? 0x4431 : 0x4420)), TagF16{});
          } else {
            const uint32_t col = j * 16 + c4 * 4;
            f = unpack16(*reinterpret_cast<const uint32_t*>(vtile + (col >> 7) * (kTileRows * 128) + swizzled_offset(row, col & 127u, 128)), Mma{});
          }
          if (see0) acc[j][0] = fmaf(p0, f.x, acc[j][0]), acc[j][1] = fmaf(p0, f.y, acc[j][1]);
          if (see1) acc[j][2] = fmaf(p1, f.x, acc[j][2]), acc[j][3] = fmaf(p1, f.y, acc[j][3]);
        }
      }
    }
  }

  __device__ __forceinline__ void sum_up() {  // the four lanes of a row meet
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
  }

  __device__ __forceinline__ void store(const PagedParams& p, const PagedUnit& u, int row0, int worker) const {
    const int lane = threadIdx.x & 31, quad = lane >> 2, c4 = lane & 3;
    const int64_t slot = (int64_t)u.index + worker;
    float* out = p.own_acc + slot * p.own_rows * D;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = row0 + h * 8 + quad;
      if (row >= u.rows) continue;
      if (c4 == 0) p.own_ml[slot * p.own_rows + row] = make_float2(m[h], l[h]);
      if constexpr (kE4M3) {
#pragma unroll
        for (int x = 0; x < D / 16; ++x)
          *reinterpret_cast<float4*>(out + row * D + x * 16 + c4 * 4) =
              make_float4(acc[2 * x][2 * h], acc[2 * x + 1][2 * h], acc[2 * x][2 * h + 1], acc[2 * x + 1][2 * h + 1]);
      } else {
#pragma unroll
        for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(out + row * D + j * 8 + c4 * 2) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
      }
    }
  }
};

// Up to eight query rows (a single token of up to eight query heads per kv head), the other way round: keys and values are the
// 16-row operand of the products, S^T = K Q^T and O^T += V^T P^T, and the query rows their eight columns, so that no half of
// a product is empty and a thread holds half as many scores, accumulators and query values: three CTAs fit on an SM instead of two
// (97 against 107 us for 32 sequences of up to 8k bf16 keys, 60 against 74 us for E4M3).  A thread has two rows (2c and
// 2c + 1), and of a tile of sixteen keys the keys quad and quad + 8 of both.
template <int D, bool kE4M3, typename QT>
struct PagedRows8 {
  using Mma = typename std::conditional<kE4M3, TagF16, QT>::type;
  static constexpr int kBoxBytes = D * (kE4M3 ? 1 : 2) < 128 ? D : 128;
  uint32_t q[D / 16][2];
  float acc[D / 16][4], scale[2], m[2], l[2];
  int limit[2];

  __device__ __forceinline__ void start(const PagedParams& p, const PagedUnit& u, int) {
    const int lane = threadIdx.x & 31, quad = lane >> 2, c4 = lane & 3;
    const bool there = quad < u.rows;
    {
      const PagedRow r = paged_row(p, u, there ? quad : 0);
      const uint8_t* src = p.q + 2 * (r.i * p.q_sb + r.h * p.q_sh + r.t * p.q_st);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        if constexpr (kE4M3) {  // four neighbours, as in a thread's codes of K
          const uint2 x = there ? *reinterpret_cast<const uint2*>(src + 2 * (k * 16 + c4 * 4)) : make_uint2(0u, 0u);
          q[k][0] = x.x, q[k][1] = x.y;
        } else {
          q[k][0] = there ? *reinterpret_cast<const uint32_t*>(src + 2 * (k * 16 + c4 * 2)) : 0u;
          q[k][1] = there ? *reinterpret_cast<const uint32_t*>(src + 2 * (k * 16 + 8 + c4 * 2)) : 0u;
        }
      }
    }
    float factor = p.scale_log2 * (kE4M3 ? p.k_scale[u.head] : 1.f);
    if constexpr (kE4M3 && std::is_same<QT, TagBf16>::value) {
      uint32_t top2 = 0u;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) top2 = absmax_bf16x2(absmax_bf16x2(top2, q[k][0]), q[k][1]);
      float top = fmaxf(__uint_as_float(top2 << 16), __uint_as_float(top2 & 0xffff0000u));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const RowShift to_f16 = row_shift(top);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) q[k][0] = bf16x2_shifted(q[k][0], to_f16), q[k][1] = bf16x2_shifted(q[k][1], to_f16);
      factor = factor / to_f16.a / to_f16.b;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // of rows 2c and 2c + 1: their lanes are 4 rows on
      const int row = 2 * c4 + e;
      scale[e] = __shfl_sync(0xffffffffu, factor, row * 4);
      limit[e] = u.key_hi - (p.T - 1 - (u.row0 + (row < u.rows ? row : 0)) / p.G);
      m[e] = -INFINITY, l[e] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  }

  template <int kKeys, int kTileRows>
  __device__ __forceinline__ void tile(const PagedUnit& u, const uint8_t* ktile, const uint8_t* vtile, int at, int key0, uint32_t valid) {
    const int lane = threadIdx.x & 31, quad = lane >> 2, c4 = lane & 3;
    const uint32_t kbase = smem_u32(ktile), vbase = smem_u32(vtile);
    constexpr uint32_t kAllValid = (1u << (kKeys / 16)) - 1u;
    const bool special = key0 < u.key_lo || key0 + kKeys > u.key_all || (valid & kAllValid) != kAllValid;
    // matrices of ldmatrix: keys 0-7 and 8-15 of a block, then of the next sixteen bytes of the row
    const uint32_t krow = at + ((lane >> 3) & 1) * 8 + (lane & 7);
    float sc[kKeys / 16][4];
#pragma unroll
    for (int j = 0; j < kKeys / 16; ++j) {
      float other[4] = {0.f, 0.f, 0.f, 0.f};  // two chains of products
      sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
      if constexpr (kE4M3) {
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
          uint32_t b[4];
          ldmatrix4(b, kbase + swizzled_offset(krow + j * 16, x * 32 + (lane >> 4) * 16, kBoxBytes));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t a[4] = {e4m3x2_to_f16x2(b[2 * e]), e4m3x2_to_f16x2(b[2 * e + 1]), e4m3x2_to_f16x2(b[2 * e] >> 16), e4m3x2_to_f16x2(b[2 * e + 1] >> 16)};
            mma16816(e ? other : sc[j], a, q[2 * x + e][0], q[2 * x + e][1], Mma{});
          }
        }
      } else {
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
          uint32_t a[4];
          const uint32_t col = x * 32 + (lane >> 4) * 16;
          ldmatrix4(a, kbase + (col >> 7) * (kTileRows * 128) + swizzled_offset(krow + j * 16, col & 127u, 128));
          mma16816(x & 1 ? other : sc[j], a, q[x][0], q[x][1], Mma{});
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[j][e] += other[e];
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < kKeys / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // row 2c + (e & 1), key quad or quad + 8
        float x = sc[j][e] * scale[e & 1];
        if (special) {
          const int key = key0 + j * 16 + (e >> 1) * 8 + quad;
          if (key < u.key_lo || key >= limit[e & 1] || !(valid >> j & 1u)) x = -INFINITY;
        }
        sc[j][e] = x;
        top[e & 1] = fmaxf(top[e & 1], x);
      }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
      top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], o));
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] + 8.f || top[1] > m[1] + 8.f)) {  // as for sixteen rows
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float next = fmaxf(m[e], top[e]);
        const float f = next == -INFINITY ? 1.f : paged_ex2(m[e] - next);
        m[e] = next;
        l[e] *= f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) acc[j][e] *= f, acc[j][e + 2] *= f;
      }
    }
    const float m0 = m[0] == -INFINITY ? 0.f : m[0], m1 = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll
    for (int j = 0; j < kKeys / 16; ++j) {
      sc[j][0] = paged_ex2(sc[j][0] - m0), sc[j][2] = paged_ex2(sc[j][2] - m0);
      sc[j][1] = paged_ex2(sc[j][1] - m1), sc[j][3] = paged_ex2(sc[j][3] - m1);
      l[0] += sc[j][0] + sc[j][2], l[1] += sc[j][1] + sc[j][3];
    }
    // values: as for sixteen rows, keys that are not there for every row are taken out of the product on both sides
#pragma unroll
    for (int kk = 0; kk < kKeys / 16; ++kk) {
      uint32_t b0 = transposed(pack16(sc[kk][0], sc[kk][1], Mma{})), b1 = transposed(pack16(sc[kk][2], sc[kk][3], Mma{}));
      uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
      if (special) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = key0 + kk * 16 + h * 8 + c4 * 2;
          const bool ok = valid >> kk & 1u;
          keep[h] = (ok && key >= u.key_lo && key < u.key_all ? 0x0000ffffu : 0u) | (ok && key + 1 >= u.key_lo && key + 1 < u.key_all ? 0xffff0000u : 0u);
        }
        b0 &= keep[0], b1 &= keep[1];
      }
      if constexpr (kE4M3) {
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {  // matrices: keys 0-7 and 8-15 of 16 codes, then of the next 16
          uint32_t b[4];
          ldmatrix4_trans(b, vbase + swizzled_offset(krow + kk * 16, x * 32 + (lane >> 4) * 16, kBoxBytes));
#pragma unroll
          for (int e = 0; e < 2; ++e) {  // (key, key + 1) x (d, d + 1) in a register: even d are rows 0-7 of the product, odd d rows 8-15
            uint32_t a[4] = {e4m3x2_to_f16x2(__byte_perm(b[2 * e], 0, 0x4420)), e4m3x2_to_f16x2(__byte_perm(b[2 * e], 0, 0x4431)),
                             e4m3x2_to_f16x2(__byte_perm(b[2 * e + 1], 0, 0x4420)), e4m3x2_to_f16x2(__byte_perm(b[2 * e + 1], 0, 0x4431))};
            if (special) a[0] &= keep[0], a[1] &= keep[0], a[2] &= keep[1], a[3] &= keep[1];
            mma16816(acc[2 * x + e], a, b0, b1, Mma{});
          }
        }
      } else {
        const uint32_t vrow = at + kk * 16 + (lane >> 4) * 8 + (lane & 7);
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {  // matrices: d 0-7 and 8-15 of keys 0-7, then of keys 8-15
          uint32_t a[4];
          const uint32_t col = x * 32 + ((lane >> 3) & 1) * 16;
          ldmatrix4_trans(a, vbase + (col >> 7) * (kTileRows * 128) + swizzled_offset(vrow, col & 127u, 128));
          if (special) a[0] &= keep[0], a[1] &= keep[0], a[2] &= keep[1], a[3] &= keep[1];
          mma16816(acc[x], a, b0, b1, Mma{});
        }
      }
    }
    if (key0 + kKeys > u.key_all) {  // the newest keys, which some rows see
#pragma unroll 1
      for (int kk = max(0, u.key_all - key0); kk < min(kKeys, u.key_hi - key0); ++kk) {
        if (!(valid >> (kk >> 4) & 1u)) continue;
        float mine[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < kKeys / 16; ++j)
          if (j == kk >> 4) mine[0] = kk & 8 ? sc[j][2] : sc[j][0], mine[1] = kk & 8 ? sc[j][3] : sc[j][1];
        const int from = (kk & 7) * 4 + c4;
        const float p0 = __shfl_sync(0xffffffffu, mine[0], from), p1 = __shfl_sync(0xffffffffu, mine[1], from);
        const bool see0 = key0 + kk < limit[0], see1 = key0 + kk < limit[1];
        const uint32_t row = at + kk;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          float2 f;  // the d of this thread's two rows of the product
          if constexpr (kE4M3) {
            const uint32_t two = *reinterpret_cast<const uint16_t*>(vtile + swizzled_offset(row, j * 16 + quad * 2, kBoxBytes));
            f = unpack16(e4m3x2_to_f16x2(two), TagF16{});
          } else {
            const uint32_t c0 = j * 32 + quad * 2, c1 = c0 + 16;
            const uint32_t lo = *reinterpret_cast<const uint16_t*>(vtile + (c0 >> 7) * (kTileRows * 128) + swizzled_offset(row, c0 & 127u, 128));
            const uint32_t hi = *reinterpret_cast<const uint16_t*>(vtile + (c1 >> 7) * (kTileRows * 128) + swizzled_offset(row, c1 & 127u, 128));
            f = unpack16(lo | hi << 16, Mma{});
          }
          if (see0) acc[j][0] = fmaf(p0, f.x, acc[j][0]), acc[j][2] = fmaf(p0, f.y, acc[j][2]);
          if (see1) acc[j][1] = fmaf(p1, f.x, acc[j][1]), acc[j][3] = fmaf(p1, f.y, acc[j][3]);
        }
      }
    }
  }

  __device__ __forceinline__ void sum_up() {  // the eight lanes of a row meet
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
      l[1] += __shfl_xor_sync(0xffffffffu, l[1], o);
    }
  }

  __device__ __forceinline__ void store(const PagedParams& p, const PagedUnit& u, int, int worker) const {
    const int lane = threadIdx.x & 31, quad = lane >> 2, c4 = lane & 3;
    const int64_t slot = (int64_t)u.index + worker;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = 2 * c4 + e;
      if (row >= u.rows) continue;
      float* out = p.own_acc + (slot * p.own_rows + row) * D;
      if (quad == 0) p.own_ml[slot * p.own_rows + row] = make_float2(m[e], l[e]);
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        if constexpr (kE4M3) *reinterpret_cast<float2*>(out + j * 16 + quad * 2) = make_float2(acc[j][e], acc[j][e + 2]);
        else out[j * 16 + quad] = acc[j][e], out[j * 16 + 8 + quad] = acc[j][e + 2];
      }
    }
  }

  // an 8 x 8 matrix of pairs (row quad, columns 2c and 2c + 1) -> its transpose in the same places
  static __device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
  }
};

// One box of tokens as a producing lane sees it: which of them a copy is asked for, and what the consumers may look at.
struct PagedBoxes {
  int tokens, per_tile;  // of a box; boxes of a tile
  __device__ __forceinline__ uint32_t valid_bits(uint32_t loads) const {  // a bit per box -> a bit per 16 keys
    const int per = tokens / 16;
    uint32_t v = 0u;
    for (int b = 0; b < per_tile; ++b)
      if (loads >> b & 1u) v |= ((1u << per) - 1u) << (b * per);
    return v;
  }
};

// Up to sixteen query rows per unit (a single token, or a few drafted ones, of a group of query heads): every warp is a worker
// with a line piece, a ring of tiles and copies of its own, and nothing in the loop waits for another warp (four warps that shared
// their tiles, as in the team below, took 25 us where this takes 12.4 and the memory 5).
template <int D, bool kE4M3, int kRows>
struct SoloSmem {
  static constexpr int kRowBytes = D * (kE4M3 ? 1 : 2);
  static constexpr int kKeys = kRowBytes == 256 ? 16 : 32;            // of a tile
  static constexpr int kTileBytes = kKeys * kRowBytes;               // K or V: 4 KB, 2 KB for E4M3 with D = 64
  static constexpr int kCtas = kRows == 8 ? 3 : 2;                   // per SM: what the registers of a row's state allow
  static constexpr int kStages = 48 * 1024 / kCtas / (2 * kTileBytes);  // 192 KB in flight per SM
  alignas(1024) uint8_t ring[4][kStages][2][kTileBytes];
  PagedSeq seq[kSmallRows];  // the plan of a small call
  int cum[kSmallRows];
  PagedLine line;
  uint64_t full[4][kStages];
  volatile uint32_t abort_flag;
  // the struct without what its alignment adds
  static constexpr int kUsed = 4 * kStages * (2 * kTileBytes + 8) + kSmallRows * ((int)sizeof(PagedSeq) + 4) + (int)sizeof(PagedLine) + 16;
};

template <int D, bool kE4M3, typename QT, int kRows>
__global__ void __launch_bounds__(128, kRows == 8 ? 3 : 2) attn_solo_kernel(const PagedParams p, const __grid_constant__ CUtensorMap map_k,
                                                           const __grid_constant__ CUtensorMap map_v) {
  using Smem = SoloSmem<D, kE4M3, kRows>;
  using Rows = typename std::conditional<kRows == 8, PagedRows8<D, kE4M3, QT>, PagedRows<D, kE4M3, QT>>::type;
  constexpr int kBytes = kE4M3 ? 1 : 2, kRowBytes = Smem::kRowBytes, kBoxBytes = kRowBytes < 128 ? kRowBytes : 128, kSubs = kRowBytes / kBoxBytes;
  constexpr int kKeys = Smem::kKeys, kStages = Smem::kStages;
  extern __shared__ __align__(1024) uint8_t raw[];
  Smem& s = *reinterpret_cast<Smem*>(raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, worker = blockIdx.x * 4 + warp;
  const bool aligned = (smem_u32(raw) & 1023u) == 0u;  // the swizzle of the tiles goes by the address
  if (threadIdx.x == 0) {
    for (int w = 0; w < 4; ++w)
      for (int i = 0; i < kStages; ++i) mbar_init(&s.full[w][i], 1);
    s.abort_flag = 0u;
    fence_barrier_init();
    fence_async_smem();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  if (p.small) {
    if (warp == 0) {
      const PagedSmall x = paged_small(p, s.cum);
      *reinterpret_cast<int4*>(s.seq + lane) = make_int4(x.slot, x.len, 0, x.cum);
      if (lane == 0) s.line = x.line;
      if (blockIdx.x == 0) {  // for the join
        if (lane < p.n) {
          int4* r = reinterpret_cast<int4*>(p.seq + lane);
          r[0] = make_int4(x.slot, x.len, 0, x.cum), r[2] = make_int4(x.left_alone, 0, 0, 0);
        }
        if (lane == 0) p.head->own = x.line;
      }
    }
    __syncthreads();
  }
  if (!aligned) {
    if (threadIdx.x == 0) p.status[1] = 99u, p.status[0] = 1u;
    return;
  }
  PagedWalk<false> ahead, walk;  // of the copies, and of the products
  ahead.start(p, worker, p.small ? PagedTables{&s.line, s.seq, s.cum} : PagedTables{&p.head->own, p.seq, p.own_cum});
  walk = ahead;
  if (walk.done()) return;

  const PagedBoxes box{min(p.c.page_tokens, kKeys), kKeys / min(p.c.page_tokens, kKeys)};
  PagedUnit next{};
  int next_tile = 0, page_base = 0, pages = 0;  // `pages`: entry page_base + lane of the table row
  bool more = true, fresh = true;
  int issued = 0;
  uint32_t valid_ring = 0u;  // two bits per stage
  auto issue = [&]() {       // asks for the tile behind the last one that was asked for
    if (!more) return;
    while (fresh || next_tile == next.tile_end) {
      if (!fresh && ahead.done()) {
        more = false;
        return;
      }
      next = ahead.next(p);
      next_tile = next.tile;
      fresh = next_tile == next.tile_end;
      if (fresh && ahead.done()) {
        more = false;
        return;
      }
      page_base = INT_MIN;
      if (!fresh) break;
    }
    const int stage = issued % kStages;
    const int first = (next_tile * kKeys) >> p.c.page_shift;
    if (page_base == INT_MIN || first + box.per_tile > page_base + 32) {
      page_base = first;
      const int at = first + lane;
      pages = at < p.c.width ? p.c.table[(int64_t)next.table_slot * p.c.table_stride + at] : -1;
    }
    // lane = box + boxes x (sub-tile + sub-tiles x (K, V))
    const int b = lane % box.per_tile, which = lane / box.per_tile;
    const int token = next_tile * kKeys + b * box.tokens;
    const int page = __shfl_sync(0xffffffffu, pages, (token >> p.c.page_shift) - page_base);
    const bool wanted = token < next.key_hi && token + box.tokens > next.key_lo && page >= 0 && page < p.c.pages;
    const uint32_t loads = __ballot_sync(0xffffffffu, wanted && which == 0);
    valid_ring = (valid_ring & ~(3u << (2 * stage))) | box.valid_bits(loads) << (2 * stage);
    if (lane == 0) mbar_expect_tx(&s.full[warp][stage], __popc(loads) * box.tokens * kRowBytes * 2);
    __syncwarp();
    if (wanted && which < 2 * kSubs) {
      const int sub = which % kSubs;
      uint8_t* dst = s.ring[warp][stage][which / kSubs] + sub * (kKeys * kBoxBytes) + b * box.tokens * kBoxBytes;
      tma_load_5d(smem_u32(dst), which / kSubs ? &map_v : &map_k, sub * (kBoxBytes / kBytes), token & (p.c.page_tokens - 1), next.head, page, p.layer,
                  &s.full[warp][stage]);
    }
    ++issued;
    ++next_tile;
  };
#pragma unroll 1
  for (int i = 0; i < kStages; ++i) issue();

  int done = 0;
  Rows rows;
  while (!walk.done()) {
    const PagedUnit u = walk.next(p);
    if (u.tile == u.tile_end) continue;
    rows.start(p, u, 0);
#pragma unroll 1
    for (int tile = u.tile; tile < u.tile_end; ++tile) {
      const int stage = done % kStages;
      if (!mbar_wait_warp(&s.full[warp][stage], (uint32_t)(done / kStages) & 1u, &s.abort_flag, p.status, 1)) {
        for (int k = done; k < issued; ++k) mbar_wait_teardown(&s.full[warp][k % kStages], (uint32_t)(k / kStages) & 1u);
        return;
      }
      rows.template tile<kKeys, kKeys>(u, s.ring[warp][stage][0], s.ring[warp][stage][1], 0, tile * kKeys, valid_ring >> (2 * stage) & 3u);
      ++done;
      __syncwarp();
      issue();
    }
    rows.sum_up();
    rows.store(p, u, 0, worker);
  }
}

// More rows than that: kWM warps side by side over rows (16 each), 4 / kWM over the keys of a tile of 64; a fifth warp asks for
// the tiles.  Bound by the products (eight warps per SM and mma.sync: 134 us for 32 rows over 537 MB of bf16).
template <int D, bool kE4M3>
struct TeamSmem {
  static constexpr int kKeys = 64;
  static constexpr int kTileBytes = kKeys * D * (kE4M3 ? 1 : 2);  // K or V of one tile
  static constexpr int kFit = 96 * 1024 / (2 * kTileBytes), kStages = kFit > 8 ? 8 : kFit;
  alignas(1024) uint8_t k[kStages][kTileBytes];
  uint8_t v[kStages][kTileBytes];
  float merge[2][16][D];
  float2 ml[4][16];
  uint64_t full[kStages], empty[kStages];
  uint32_t valid[kStages];  // a bit per 16 keys: the table names a page of the pool
  volatile uint32_t abort_flag;
  static constexpr int kUsed = kStages * (2 * kTileBytes + 16 + 4) + 2 * 16 * D * 4 + 4 * 16 * 8 + 16;
};

template <int D, bool kE4M3, typename QT, int kWM>
__global__ void __launch_bounds__(160, 2) attn_team_kernel(const PagedParams p, const __grid_constant__ CUtensorMap map_k,
                                                           const __grid_constant__ CUtensorMap map_v) {
  using Smem = TeamSmem<D, kE4M3>;
  constexpr int kBytes = kE4M3 ? 1 : 2, kRowBytes = D * kBytes, kBoxBytes = kRowBytes < 128 ? kRowBytes : 128, kSubs = kRowBytes / kBoxBytes;
  constexpr int kTile = Smem::kKeys, kWK = 4 / kWM, kKeys = kTile / kWK;  // keys of a tile that one warp takes
  constexpr int kStages = Smem::kStages;
  extern __shared__ __align__(1024) uint8_t raw[];
  Smem& s = *reinterpret_cast<Smem*>(raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool aligned = (smem_u32(raw) & 1023u) == 0u;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&s.full[i], 1), mbar_init(&s.empty[i], 4);
    s.abort_flag = 0u;
    fence_barrier_init();
    fence_async_smem();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  if (!aligned) {
    if (threadIdx.x == 0) p.status[1] = 99u, p.status[0] = 1u;
    return;
  }
  PagedWalk<false> walk;
  walk.start(p, blockIdx.x, {&p.head->own, p.seq, p.own_cum});

  if (warp == 4) {  // ---- producer: lane b of a tile's boxes asks for its own part of the pages
    const PagedBoxes box{min(p.c.page_tokens, kTile), kTile / min(p.c.page_tokens, kTile)};
    int stage = 0, issued = 0;
    uint32_t parity = 1u;
    while (!walk.done()) {
      const PagedUnit u = walk.next(p);
      const int32_t* row = p.c.table + (int64_t)u.table_slot * p.c.table_stride;
      for (int tile = u.tile; tile < u.tile_end; ++tile) {
        const int token = tile * kTile + lane * box.tokens;
        const bool wanted = lane < box.per_tile && token < u.key_hi && token + box.tokens > u.key_lo;
        int page = -1;
        if (wanted) page = row[token >> p.c.page_shift];
        const bool load = wanted && page >= 0 && page < p.c.pages;
        const uint32_t loads = __ballot_sync(0xffffffffu, load);
        const bool go = mbar_wait_warp(&s.empty[stage], parity, &s.abort_flag, p.status, 1);
        if (lane == 0) {
          s.valid[stage] = box.valid_bits(loads);
          mbar_expect_tx(&s.full[stage], go ? __popc(loads) * box.tokens * kRowBytes * 2 : 0);
        }
        __syncwarp();
        if (go && load) {
          const int in_page = token & (p.c.page_tokens - 1);
#pragma unroll
          for (int x = 0; x < kSubs; ++x) {
            const uint32_t off = x * (kTile * kBoxBytes) + lane * box.tokens * kBoxBytes;
            tma_load_5d(smem_u32(s.k[stage]) + off, &map_k, x * (kBoxBytes / kBytes), in_page, u.head, page, p.layer, &s.full[stage]);
            tma_load_5d(smem_u32(s.v[stage]) + off, &map_v, x * (kBoxBytes / kBytes), in_page, u.head, page, p.layer, &s.full[stage]);
          }
        }
        ++issued;
        if (++stage == kStages) stage = 0, parity ^= 1u;
      }
    }
    if (s.abort_flag)  // copies in flight land before the CTA leaves
      for (int k = max(0, issued - kStages); k < issued; ++k) mbar_wait_teardown(&s.full[k % kStages], (uint32_t)(k / kStages) & 1u);
    return;
  }

  // ---- consumers
  const int wm = warp % kWM, wk = warp / kWM, quad = lane >> 2, c4 = lane & 3;
  int stage = 0;
  uint32_t parity = 0u;
  PagedRows<D, kE4M3, QT> rows;
  while (!walk.done()) {
    const PagedUnit u = walk.next(p);
    if (u.tile == u.tile_end) continue;
    rows.start(p, u, wm * 16);
    for (int tile = u.tile; tile < u.tile_end; ++tile) {
      mbar_wait_warp(&s.full[stage], parity, &s.abort_flag, p.status, 2);
      rows.template tile<kKeys, kTile>(u, s.k[stage], s.v[stage], wk * kKeys, tile * kTile + wk * kKeys, s.valid[stage] >> (wk * kKeys / 16));
      mbar_arrive_warp(&s.empty[stage]);
      if (++stage == kStages) stage = 0, parity ^= 1u;
    }
    rows.sum_up();
    if constexpr (kWK > 1) {  // the warps over keys meet: the upper half of them hands its sums to the lower half
      if (c4 == 0) s.ml[warp][quad] = make_float2(rows.m[0], rows.l[0]), s.ml[warp][quad + 8] = make_float2(rows.m[1], rows.l[1]);
      asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 x = s.ml[warp][quad + 8 * h], y = s.ml[(wk ^ 1) * kWM + wm][quad + 8 * h];
        const float top = fmaxf(x.x, y.x);
        const float f = x.x == -INFINITY ? 0.f : paged_ex2(x.x - top), g = y.x == -INFINITY ? 0.f : paged_ex2(y.x - top);
        rows.m[h] = top, rows.l[h] = x.y * f + y.y * g;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) rows.acc[j][2 * h] *= f, rows.acc[j][2 * h + 1] *= f;
      }
      float* buf = &s.merge[wm][0][0];
      if (wk == 1) {
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          *reinterpret_cast<float2*>(buf + quad * D + j * 8 + c4 * 2) = make_float2(rows.acc[j][0], rows.acc[j][1]);
          *reinterpret_cast<float2*>(buf + (quad + 8) * D + j * 8 + c4 * 2) = make_float2(rows.acc[j][2], rows.acc[j][3]);
        }
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (wk == 0) {
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          const float2 x = *reinterpret_cast<const float2*>(buf + quad * D + j * 8 + c4 * 2);
          const float2 y = *reinterpret_cast<const float2*>(buf + (quad + 8) * D + j * 8 + c4 * 2);
          rows.acc[j][0] += x.x, rows.acc[j][1] += x.y, rows.acc[j][2] += y.x, rows.acc[j][3] += y.y;
        }
      }
    }
    if (wk == 0) rows.store(p, u, wm * 16, blockIdx.x);
  }
}

// ---- join -------------------------------------------------------------------------------------------------------------
// One warp per output row, or (kSplit) four, each with a quarter of the pieces and sums of its own, where the rows are few (one
// sequence of 8k keys has 128 pieces a row: 1.7 us less of a call of 16.7 than when the four went through them together, 32
// at a time).  The statistics of 32 pieces come to the lanes at once, so that what is left to wait for is one round of loads: a
// lane holds D / 32 neighbours of eight pieces at a time (one piece behind another took 26 us where this takes 12, and 3 to 5 with
// four warps).  Latency bounds it, and for many rows the memory (16384 rows of 5 to 7 pieces: 18 us).  Which pieces there are
// follows from the plan, which is read behind this launch's own wait: the plan has ended when the launch comes up, but only the wait
// makes what earlier launches wrote visible.
template <int D, typename QT, bool kSplit>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedParams p) {
  constexpr int kPer = D / 32;
  __shared__ float parts[kSplit ? 3 : 1][D];
  __shared__ float2 part_ml[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = kSplit ? warp : 0;
  const uint32_t w = kSplit ? blockIdx.x : blockIdx.x * 4 + warp;
  pdl_trigger();
  const bool there = w < (uint32_t)(p.n * p.Hq * p.T);
  const uint32_t row_id = there ? w : 0u;
  const uint32_t t = p.T == 1 ? 0u : row_id % (uint32_t)p.T, ih = p.T == 1 ? row_id : row_id / (uint32_t)p.T, i = ih / (uint32_t)p.Hq, h = ih - i * (uint32_t)p.Hq;
  pdl_wait();
  const PagedSeq s = p.seq[i];
  const PagedHead line = *p.head;
  const int head = h / (uint32_t)p.G, r = t * p.G + (h - head * p.G), len = s.len;
  float acc[kPer], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
  // the workers that have a part of the unit's tiles: from the one where the first tile lies to the one where the last does
  int n_prefix = 0, prefix_row = 0, n_own = 0, own_row = 0, two = 0;
  int64_t prefix_slot = 0, own_slot = 0;
  if (len - (p.T - 1 - (int)t) > 0) {
    if (s.first > 0) {
      const int row = ((int)i - s.g_row) * p.R + r, block = row >> p.prefix_shift, which = head * s.g_blocks + block;
      const int tiles = (s.first + kPagedPrefixTile - 1) / kPagedPrefixTile;
      const PagedCut cut = line.prefix.cut;
      const uint32_t from = s.g_cum + which * cut.length(tiles) + cut.extra, worker = from / cut.per;
      two = prefix_in_two(p, s.g_rows - (block << p.prefix_shift));
      n_prefix = (int)((from + tiles - 1) / cut.per - worker + 1) << two;
      prefix_slot = s.g_unit + which + (int64_t)worker;
      prefix_row = row & (p.prefix_rows - 1);
    }
    const int block = r >> p.own_rows_shift, which = head * p.own_blocks + block, tiles = own_tiles(p, s.first, len);
    const PagedCut cut = line.own.cut;
    const uint32_t from = s.cum * p.own_units + which * cut.length(tiles) + cut.extra, worker = from / cut.per;
    own_slot = (int64_t)i * p.own_units + which + worker;
    n_own = (int)((from + tiles - 1) / cut.per - worker) + 1;
    own_row = r & (p.own_rows - 1);
  }
  if (!there) return;
  auto o_at = [&]() { return p.o + 2 * ((int64_t)i * p.o_sb + (int64_t)h * p.o_sh + (int64_t)t * p.o_st + lane * kPer); };
  auto lse_at = [&]() { return p.lse + ((int64_t)i * p.Hq + h) * p.T + t; };
  if (s.left_alone) {  // in no group; the same for all warps of a row
    if (p.flags & FA4B_PAGED_CLEAR_O) {
      if constexpr (kPer == 4) *reinterpret_cast<uint2*>(o_at()) = make_uint2(0u, 0u);
      else *reinterpret_cast<uint32_t*>(o_at()) = 0u;
    }
    if (lane == 0 && (p.flags & FA4B_PAGED_CLEAR_LSE)) *lse_at() = -INFINITY;
    return;
  }
  const int total = n_prefix + n_own, each = kSplit ? (total + 3) / 4 : total, end = min(total, (part + 1) * each);
  for (int base = part * each; base < end; base += 32) {
    const int k = base + lane;
    const bool is_prefix = k < n_prefix;
    const int64_t row = is_prefix ? (prefix_slot + (k >> two)) * p.prefix_rows + (k & two) * 64 + prefix_row : (own_slot + (k - n_prefix)) * p.own_rows + own_row;
    float2 x = make_float2(-INFINITY, 0.f);
    if (k < end) x = is_prefix ? p.prefix_ml[row] : p.own_ml[row];
    float top = x.x;
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float next = fmaxf(m, top), f = m == -INFINITY ? 0.f : paged_ex2(m - next);
    const float y = x.x == -INFINITY ? 0.f : paged_ex2(x.x - next);
    float sum = x.y * y;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    m = next, l = l * f + sum;
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] *= f;
    const float* at = (is_prefix ? p.prefix_acc : p.own_acc) + row * D;
    const int count = min(32, end - base);
    for (int k0 = 0; k0 < count; k0 += 8) {
      float v[8][kPer], weight[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        weight[j] = __shfl_sync(0xffffffffu, y, (k0 + j) & 31);
        const float* from_row = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, (unsigned long long)at, (k0 + j) & 31));
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[j][e] = 0.f;
        if (k0 + j < count) {
          if constexpr (kPer == 4) {
            const float4 q = __ldcg(reinterpret_cast<const float4*>(from_row) + lane);
            v[j][0] = q.x, v[j][1] = q.y, v[j][2] = q.z, v[j][3] = q.w;
          } else {
            const float2 q = __ldcg(reinterpret_cast<const float2*>(from_row) + lane);
            v[j][0] = q.x, v[j][1] = q.y;
          }
        } else {
          weight[j] = 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < kPer; ++e) acc[e] = fmaf(v[j][e], weight[j], acc[e]);
    }
  }
  if constexpr (kSplit) {
    if (warp > 0) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) parts[warp - 1][lane * kPer + e] = acc[e];
    }
    if (lane == 0) part_ml[warp] = make_float2(m, l);
    __syncthreads();
    if (warp > 0) return;
    const float top = fmaxf(fmaxf(m, part_ml[1].x), fmaxf(part_ml[2].x, part_ml[3].x)), f = m == -INFINITY ? 0.f : paged_ex2(m - top);
    m = top, l *= f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] *= f;
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float2 x = part_ml[w];
      const float g = x.x == -INFINITY ? 0.f : paged_ex2(x.x - top);
      l = fmaf(x.y, g, l);
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] = fmaf(parts[w - 1][lane * kPer + e], g, acc[e]);
    }
  }
  const float inv = l == 0.f ? 0.f : (p.v_scale ? p.v_scale[head] : 1.f) / l;  // a row that sees nothing: zeros, -inf
  uint8_t* out = o_at();
  if constexpr (kPer == 4) *reinterpret_cast<uint2*>(out) = make_uint2(pack16(acc[0] * inv, acc[1] * inv, QT{}), pack16(acc[2] * inv, acc[3] * inv, QT{}));
  else *reinterpret_cast<uint32_t*>(out) = pack16(acc[0] * inv, acc[1] * inv, QT{});
  if (lane == 0) *lse_at() = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

}  // namespace fa4b

// ---- host -------------------------------------------------------------------------------------------------------------
namespace fa4b {

struct PagedMaps {
  CUtensorMap own_k, own_v, prefix_k, prefix_v;
};

template <typename Smem, typename K>
static int launch_units(K kernel, const PagedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, int ctas, int threads, cudaStream_t st,
                        std::atomic<uint64_t>& allowed) {
  constexpr int smem = Smem::kUsed;
  static_assert(smem >= (int)offsetof(Smem, abort_flag) + 4 && smem <= 113 * 1024, "two CTAs per SM");
  if (int s = allow_smem(kernel, smem, allowed)) return s;
  FA4B_CUDA(launch_overlapped(kernel, ctas, threads, smem, st, p, mk, mv));
  return FA4B_OK;
}

template <int D, bool kE4M3, typename QT>
static int launch_paged(const PagedParams& p, const PagedMaps& m, cudaStream_t st) {
  const size_t smem = 4 * paged_plan_words(p.n, p.groups);
  static std::atomic<uint64_t> allowed[5];
  if (smem > kSmemUnasked)
    if (int s = allow_smem(paged_plan_kernel, 4 * (int)paged_plan_words(kPagedMaxRows, kPagedMaxRows), allowed[3])) return s;
  if (!p.small) FA4B_CUDA(launch_overlapped(paged_plan_kernel, 1, kPlanThreads, smem, st, p));
  if (p.groups > 0)
    if (int s = launch_prefix(p, D, kE4M3, std::is_same<QT, TagF16>::value, m.prefix_k, m.prefix_v, st)) return s;
  // which of these a type takes: see paged_params
  int s;
  if (p.own_rows == 8) s = launch_units<SoloSmem<D, kE4M3, 8>>(attn_solo_kernel<D, kE4M3, QT, 8>, p, m.own_k, m.own_v, p.own_workers / 4, 128, st, allowed[4]);
  else if (p.own_rows == 16) s = launch_units<SoloSmem<D, kE4M3, 16>>(attn_solo_kernel<D, kE4M3, QT, 16>, p, m.own_k, m.own_v, p.own_workers / 4, 128, st, allowed[0]);
  else if constexpr (kE4M3 && D == 128) s = FA4B_UNSUPPORTED;
  else if (p.own_rows == 32) s = launch_units<TeamSmem<D, kE4M3>>(attn_team_kernel<D, kE4M3, QT, 2>, p, m.own_k, m.own_v, p.own_workers, 160, st, allowed[1]);
  else if constexpr (!kE4M3 && D == 64) s = FA4B_UNSUPPORTED;
  else s = launch_units<TeamSmem<D, kE4M3>>(attn_team_kernel<D, kE4M3, QT, 4>, p, m.own_k, m.own_v, p.own_workers, 160, st, allowed[2]);
  if (s) return s;
  const int64_t rows = (int64_t)p.n * p.Hq * p.T;
  // four warps a row up to where the rows alone fill the SMs with warps, 8 CTAs of four each (1024 rows: 5.7 against 7.0 us; 1536 rows:
  // 5.8 against 3.5 us)
  if (rows <= 8ll * p.prefix_workers) FA4B_CUDA(launch_overlapped(paged_join_kernel<D, QT, true>, (unsigned)rows, 128, 0, st, p));
  else FA4B_CUDA(launch_overlapped(paged_join_kernel<D, QT, false>, (unsigned)((rows + 3) / 4), 128, 0, st, p));
  return FA4B_OK;
}

// checks a call and lays its workspace out; `ws` may be NULL (a size query)
static int paged_params(const fa4b_kv_cache* c, const fa4b_attn_paged_args* a, PagedParams* out, size_t* bytes) {
  PagedParams p{};
  if (int s = kv_view(c, &p.c)) return s;
  FA4B_REQUIRE(a != nullptr, FA4B_BAD_ARG, "args is NULL");
  FA4B_REQUIRE(a->n >= 0 && a->n <= kPagedMaxRows, FA4B_BAD_SHAPE, "n=%d: batches of 0 to %d rows are built", a->n, kPagedMaxRows);
  FA4B_REQUIRE(a->T >= 1 && a->T <= kPagedMaxT, FA4B_BAD_SHAPE, "T=%d: 1 to %d query tokens per sequence are built", a->T, kPagedMaxT);
  FA4B_REQUIRE(a->Hq > 0 && a->Hq % c->Hkv == 0, FA4B_BAD_SHAPE, "Hq=%d must be a multiple of Hkv=%d", a->Hq, c->Hkv);
  FA4B_REQUIRE((int64_t)a->n * a->Hq * a->T < INT32_MAX, FA4B_BAD_SHAPE, "n Hq T must be below 2^31");
  FA4B_REQUIRE(a->Hq / c->Hkv <= 128, FA4B_BAD_SHAPE, "%d query heads per kv head: at most 128 are built", a->Hq / c->Hkv);
  FA4B_REQUIRE(a->layer >= 0 && a->layer < c->layers, FA4B_BAD_SHAPE, "layer %d of %d", a->layer, c->layers);
  FA4B_REQUIRE(a->q_dtype == FA4B_KV_BF16 || a->q_dtype == FA4B_KV_F16, FA4B_UNSUPPORTED, "queries are bf16 or f16");
  FA4B_REQUIRE(c->dtype == FA4B_KV_E4M3 || a->q_dtype == c->dtype, FA4B_UNSUPPORTED, "a 16-bit cache takes queries of its own type");
  FA4B_REQUIRE(a->groups >= 0 && a->groups <= std::max(a->n, 1), FA4B_BAD_SHAPE, "groups=%d: at most one for each of %d rows", a->groups, a->n);
  FA4B_REQUIRE(a->groups == 0 || (a->group_offsets && a->shared_lens), FA4B_BAD_ARG, "groups need group_offsets and shared_lens");
  FA4B_REQUIRE((a->flags & ~(FA4B_PAGED_CLEAR_O | FA4B_PAGED_CLEAR_LSE)) == 0, FA4B_BAD_ARG, "unknown flags 0x%x", a->flags);
  FA4B_REQUIRE(a->seqs || a->n <= c->max_seqs, FA4B_BAD_SHAPE, "n=%d rows without a list of slots, and %d slots", a->n, c->max_seqs);
  p.layer = a->layer, p.n = a->n, p.T = a->T, p.Hq = a->Hq, p.G = a->Hq / c->Hkv, p.R = p.T * p.G, p.groups = a->groups, p.flags = a->flags;
  p.seqs = a->seqs, p.offsets = a->group_offsets, p.shared = a->shared_lens;
  p.q = static_cast<const uint8_t*>(a->q), p.q_sb = a->q_strides.batch, p.q_sh = a->q_strides.head, p.q_st = a->q_strides.seq;
  p.o = static_cast<uint8_t*>(a->o), p.o_sb = a->o_strides.batch, p.o_sh = a->o_strides.head, p.o_st = a->o_strides.seq;
  p.lse = a->lse;
  for (int64_t s : {p.q_sb, p.q_sh, p.q_st, p.o_sb, p.o_sh, p.o_st})
    FA4B_REQUIRE(s % 8 == 0, FA4B_BAD_ALIGN, "strides of q and o must be multiples of 8 elements");
  FA4B_REQUIRE((p.n <= 1 || p.o_sb != 0) && (p.Hq == 1 || p.o_sh != 0) && (p.T == 1 || p.o_st != 0), FA4B_BAD_SHAPE, "rows of o lie on one another (a stride of 0)");
  FA4B_REQUIRE(!misaligned(p.q, 16) && !misaligned(p.o, 16), FA4B_BAD_ALIGN, "q and o must be 16-byte aligned");
  FA4B_REQUIRE(std::isfinite(a->softmax_scale), FA4B_BAD_ARG, "softmax_scale is not a finite number");
  p.scale_log2 = (a->softmax_scale > 0.f ? a->softmax_scale : 1.0f / sqrtf((float)c->D)) * kLog2e;
  if (c->dtype == FA4B_KV_E4M3) p.k_scale = c->k_scale + (int64_t)a->layer * c->Hkv, p.v_scale = c->v_scale + (int64_t)a->layer * c->Hkv;
  const int n_sm = sm_count() > 0 ? sm_count() : 148;
  // Rows of an own unit.  32 sequences of up to 8k keys, 8 kv heads (us; rows of a sequence and kv head on the left):
  //   bf16 D 128   8: 8 rows 97, 16 rows 107, 32 rows 120     16: 16 rows 109, 32 rows 124      32: 16 rows 187, 32 rows 134, 64 rows 212
  //   56 (4 kv heads): 16 rows 162, 32 rows 123, 64 rows 120
  //   E4M3 D 128   8: 8 rows 60, 16 rows 74     16: 16 rows 78, 32 rows 151     32: 16 rows 145, 32 rows 161     56: 16 rows 141, 64 rows 146
  //   bf16 D 64   32: 16 rows 104, 32 rows 87      56: 32 rows 86, 64 rows 90       E4M3 D 64   32: 16 rows 110, 32 rows 94      56: 32 rows 92, 64 rows 82
  // With E4M3 and D = 128 a warp spends as long on turning codes as on products, and the warps of a team all turn the same ones.
  const bool wide_codes = c->dtype == FA4B_KV_E4M3 && c->D == 128, short_16 = c->dtype != FA4B_KV_E4M3 && c->D == 64;
  p.own_rows = p.R <= 8 ? 8 : p.R <= 16 || wide_codes ? 16 : p.R <= 32 || short_16 ? 32 : 64;
  p.own_blocks = (p.R + p.own_rows - 1) / p.own_rows;
  const bool solo = p.own_rows <= 16, short_rows = c->D * (c->dtype == FA4B_KV_E4M3 ? 1 : 2) < 256;
  p.own_tile = !solo ? TeamSmem<64, true>::kKeys : short_rows ? 32 : 16;
  p.own_shift = __builtin_ctz((unsigned)p.own_tile), p.own_rows_shift = __builtin_ctz((unsigned)p.own_rows), p.own_units = c->Hkv * p.own_blocks;
  p.own_workers = (p.own_rows == 8 ? 12 : solo ? 8 : 2) * n_sm;
  p.own_extra = solo ? 2 : 1;
  p.own_min = solo ? 64 / p.own_tile : 1;  // a piece shorter than 64 keys is mostly its beginning
  // Two blocks of 128 rows over the same keys where the groups have the rows for it: each tile then comes from memory half as
  // often (8 groups of 160 rows over 8k keys: bf16 D 128 99 against 135 us, E4M3 108 against 125, D 64 83 against 91 and 94
  // against 97).  With fewer rows the two halves of a CTA take the keys in turn (8 groups of 128 rows: E4M3 83 against 86 us,
  // D 64 61 against 67; 8 groups of 16 rows over 32k keys: 172 against 197 and 99 against 155); but bf16 with D = 128 is bound by the
  // tensor core's 64-key products either way and better off without the join of the halves (83 against 87 us; 207 against 215).
  p.prefix_rows = p.groups > 0 && ((int64_t)p.n * p.R > 128ll * p.groups || paged_prefix_wide(c->D, c->dtype == FA4B_KV_E4M3)) ? 256 : 128;
  p.prefix_shift = __builtin_ctz((unsigned)p.prefix_rows), p.prefix_workers = n_sm, p.prefix_extra = 3;
  p.small = p.groups == 0 && p.n <= kSmallRows && solo;
  const int64_t keys = (int64_t)c->table_width * c->page_tokens, own_length = 2 * (keys / p.own_tile) + 2 + p.own_extra;
  const int64_t prefix_units = p.groups ? (int64_t)c->Hkv * (((int64_t)p.n * p.R + p.prefix_rows - 1) / p.prefix_rows + p.groups) : 0;
  const int64_t own_slots = (int64_t)p.n * c->Hkv * p.own_blocks + p.own_workers, prefix_slots = p.groups ? prefix_units + p.prefix_workers : 0;
  // positions on the lines (of one head and row block, and of all) are counted in 32 bits
  FA4B_REQUIRE(p.n * own_length < INT32_MAX && prefix_units * (2 * (keys / kPagedPrefixTile) + 2 + p.prefix_extra) < INT32_MAX && own_slots < INT32_MAX, FA4B_BAD_SHAPE,
               "%d rows over tables of %d pages of %d tokens are too many for one call", p.n, c->table_width, c->page_tokens);
  size_t off = 0;
  uint8_t* ws = static_cast<uint8_t*>(a->ws);
  auto take = [&](size_t size) {
    uint8_t* at = ws ? ws + off : nullptr;
    off = align_up(off + size, 256);
    return at;
  };
  const size_t n = p.n, g = p.groups;
  p.head = reinterpret_cast<PagedHead*>(take(sizeof(PagedHead)));
  p.seq = reinterpret_cast<PagedSeq*>(take(sizeof(PagedSeq) * n));
  p.group = reinterpret_cast<PagedGroup*>(take(sizeof(PagedGroup) * g));
  p.own_cum = reinterpret_cast<int*>(take(4 * n));
  p.g_cum = reinterpret_cast<int*>(take(4 * g));
  p.own_ml = reinterpret_cast<float2*>(take((size_t)own_slots * p.own_rows * 8));
  p.prefix_ml = reinterpret_cast<float2*>(take((size_t)prefix_slots * p.prefix_rows * 8));
  p.own_acc = reinterpret_cast<float*>(take((size_t)own_slots * p.own_rows * c->D * 4));
  p.prefix_acc = reinterpret_cast<float*>(take((size_t)prefix_slots * p.prefix_rows * c->D * 4));
  p.status = reinterpret_cast<uint32_t*>(p.c.work + kKvAttnStatus);
  *out = p;
  *bytes = off;
  return FA4B_OK;
}

}  // namespace fa4b

using namespace fa4b;

extern "C" {

size_t fa4b_attn_paged_workspace_bytes(const fa4b_kv_cache* c, const fa4b_attn_paged_args* a) {
  PagedParams p;
  size_t bytes = 0;
  return paged_params(c, a, &p, &bytes) == FA4B_OK ? bytes : 0;
}

int fa4b_attn_paged_fwd(const fa4b_kv_cache* c, const fa4b_attn_paged_args* a, void* stream) {
  PagedParams p;
  size_t bytes = 0;
  if (int s = paged_params(c, a, &p, &bytes)) return s;
  if (a->n == 0) return FA4B_OK;
  FA4B_REQUIRE(a->q && a->o && a->lse && a->ws, FA4B_BAD_ARG, "q, o, lse or ws is NULL");
  FA4B_REQUIRE(!misaligned(a->ws, 256), FA4B_BAD_ALIGN, "ws must be 256-byte aligned");
  const bool e4m3 = c->dtype == FA4B_KV_E4M3;
  // one map per pool and width of a copy: the units take what a tile of theirs holds of a page
  const int esz = e4m3 ? 1 : 2;
  const uint64_t dims[5] = {(uint64_t)c->D, (uint64_t)c->page_tokens, (uint64_t)c->Hkv, (uint64_t)c->num_pages, (uint64_t)c->layers};
  const uint64_t sk[4] = {(uint64_t)p.c.row_bytes, (uint64_t)p.c.row_bytes * c->page_tokens, (uint64_t)p.c.k_page, (uint64_t)p.c.k_layer};
  const uint64_t sv[4] = {sk[0], sk[1], (uint64_t)p.c.v_page, (uint64_t)p.c.v_layer};
  uint32_t box[5] = {(uint32_t)std::min(c->D, 128 / esz), (uint32_t)std::min(c->page_tokens, p.own_tile), 1, 1, 1};
  PagedMaps m;
  if (int s = make_tensor_map_5d(&m.own_k, c->k, esz, dims, sk, box)) return s;
  if (int s = make_tensor_map_5d(&m.own_v, c->v, esz, dims, sv, box)) return s;
  m.prefix_k = m.own_k, m.prefix_v = m.own_v;
  if (p.groups > 0 && (int)box[1] != std::min(c->page_tokens, kPagedBox)) {
    box[1] = (uint32_t)std::min(c->page_tokens, kPagedBox);
    if (int s = make_tensor_map_5d(&m.prefix_k, c->k, esz, dims, sk, box)) return s;
    if (int s = make_tensor_map_5d(&m.prefix_v, c->v, esz, dims, sv, box)) return s;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool q16 = a->q_dtype == FA4B_KV_F16;
  if (c->D == 128) {
    if (e4m3) return q16 ? launch_paged<128, true, TagF16>(p, m, st) : launch_paged<128, true, TagBf16>(p, m, st);
    return q16 ? launch_paged<128, false, TagF16>(p, m, st) : launch_paged<128, false, TagBf16>(p, m, st);
  }
  if (e4m3) return q16 ? launch_paged<64, true, TagF16>(p, m, st) : launch_paged<64, true, TagBf16>(p, m, st);
  return q16 ? launch_paged<64, false, TagF16>(p, m, st) : launch_paged<64, false, TagBf16>(p, m, st);
}

}  // extern "C"
