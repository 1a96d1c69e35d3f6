// Attention of the newest tokens of a batch over a paged cache (single tokens, or a few drafted ones), with the keys that
// a group of sequences shares read once for all of them.
//
// Bound by memory: a key and a value are used by the few query rows of one sequence (own units), so the kernel is a
// stream of pages through shared memory: one warp asks for tiles of 64 keys by TMA several tiles ahead, four warps
// consume them.  Scores and values go through mma.sync m16n8k16: with 4 to 16 query rows a tcgen05 tile of 128 rows would
// be empty for the most part, and the 16-row form already computes a tile in a quarter of the time its bytes take.
#include "attn_paged.cuh"

#include <type_traits>

namespace fa4b {

constexpr int kPagedThreads = 160;
constexpr int kPagedStageBytes = 96 * 1024;  // shared memory for tiles in flight; two CTAs per SM

// ---- plan -------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int paged_scan(int v, int* warp_sums, int& total) {  // exclusive, 1024 threads
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int w = warp_sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  __syncthreads();
  return x - v + (warp ? before : 0);
}

// One CTA: lengths, groups, and the lines of tiles.  The shared part of a group is what the caller says, cut to what every
// query row of every member sees (so that no row of a prefix unit needs a mask) and to whole 16 keys; a group of one
// member has none.
__global__ void __launch_bounds__(1024) paged_plan_kernel(const PagedParams p) {
  __shared__ int warp_sums[32];
  extern __shared__ int dyn[];
  int* g_min = dyn;              // [groups] shortest member's length - T
  int* g_first = dyn + p.groups;
  int* g_count = dyn + 2 * p.groups;
  pdl_trigger();
  for (int g = threadIdx.x; g < p.groups; g += 1024) g_min[g] = INT_MAX, g_first[g] = INT_MAX, g_count[g] = 0;
  pdl_wait();
  bool bad = false;  // groups have to lie behind one another: the slots of their units are counted on it
  for (int g = threadIdx.x; g < p.groups; g += 1024) bad |= p.offsets[g] < 0 || p.offsets[g + 1] < p.offsets[g] || p.offsets[g + 1] > p.n;
  bad = __syncthreads_or(bad);
  if (bad && threadIdx.x == 0 && atomicCAS(p.status, 0u, 2u) == 0u) p.status[1] = (uint32_t)p.groups;
  for (int i = threadIdx.x; i < p.n; i += 1024) {
    const int slot = p.seqs ? p.seqs[i] : i;
    int len = 0, g = p.groups > 0 || bad ? -1 : 0;
    if (slot >= 0 && slot < p.c.max_seqs) len = (int)min((int64_t)max(p.c.lens[slot], 0), (int64_t)p.c.width << p.c.page_shift);
    if (p.groups > 0 && !bad) {
      int lo = 0, hi = p.groups;  // the last group that begins at or before i
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.offsets[mid] <= i) lo = mid; else hi = mid - 1;
      }
      if (lo < p.groups && p.offsets[lo] <= i && i < p.offsets[lo + 1]) g = lo;
    }
    p.plan.slot[i] = slot, p.plan.len[i] = len, p.plan.group[i] = g;
    if (p.groups > 0 && g >= 0 && len > 0) {
      atomicMin(g_min + g, max(len - p.T, 0));
      atomicMin(g_first + g, i);
      atomicAdd(g_count + g, 1);
    }
  }
  __syncthreads();
  for (int g = threadIdx.x; g < p.groups; g += 1024) {
    g_min[g] = g_count[g] > 1 ? min(max(p.shared[g], 0), g_min[g]) / kPagedAlign * kPagedAlign : 0;
    g_count[g] = 0;
  }
  __syncthreads();
  // A shared page that the table does not name: the group goes without, the own units know how to leave such a page out.
  const int per_group = 1024 >> (32 - __clz(min(max(p.groups, 1), 32) - 1));  // threads: a warp at least
  for (int g = threadIdx.x / per_group; g < p.groups; g += 1024 / per_group) {
    const int pages = (g_min[g] + p.c.page_tokens - 1) >> p.c.page_shift;
    const int32_t* row = p.c.table + (pages ? (int64_t)p.plan.slot[g_first[g]] * p.c.table_stride : 0);
    bool missing = false;
    for (int j = threadIdx.x % per_group; j < pages; j += per_group) missing |= (uint32_t)row[j] >= (uint32_t)p.c.pages;
    if (missing) g_count[g] = 1;
  }
  __syncthreads();
  int tiles = 0, units = 0;
  for (int base = 0; base < p.groups; base += 1024) {
    const int g = base + threadIdx.x;
    int own_t = 0, own_u = 0;
    if (g < p.groups) {
      const int lo = max(p.offsets[g], 0), hi = min(p.offsets[g + 1], p.n);
      const int shared = hi <= lo || bad || g_count[g] ? 0 : g_min[g];
      own_u = hi > lo && !bad ? p.c.heads * ceil_div((hi - lo) * p.R, p.prefix_rows) : 0;
      own_t = own_u * ceil_div(shared, p.prefix_tile);
      p.plan.g_shared[g] = shared;
      p.plan.g_first[g] = shared ? g_first[g] : 0;
      g_min[g] = shared;
    }
    int t_total, u_total;
    const int t_before = paged_scan(own_t, warp_sums, t_total), u_before = paged_scan(own_u, warp_sums, u_total);
    if (g < p.groups) p.plan.g_cum[g] = tiles + t_before, p.plan.g_unit[g] = units + u_before;
    tiles += t_total, units += u_total;
  }
  if (threadIdx.x == 0) p.plan.g_cum[p.groups] = tiles, p.plan.g_unit[p.groups] = units;
  __syncthreads();
  tiles = 0;
  for (int base = 0; base < p.n; base += 1024) {
    const int i = base + threadIdx.x;
    int t = 0;
    if (i < p.n) {
      const int g = p.plan.group[i];
      if (g >= 0) t = own_tiles(p.groups > 0 ? g_min[g] : 0, p.plan.len[i]);
    }
    int total;
    const int before = paged_scan(t, warp_sums, total);
    if (i < p.n) p.plan.own_cum[i] = tiles + before;
    tiles += total;
  }
  if (threadIdx.x == 0) p.plan.own_cum[p.n] = tiles;
}

// ---- the units over keys of one sequence ----------------------------------------------------------------------------------
template <int D, int kBytes>
struct PagedSmem {
  static constexpr int kTileBytes = kPagedTile * D * kBytes;  // K or V of one tile
  static constexpr int kStages = kPagedStageBytes / (2 * kTileBytes) > 8 ? 8 : kPagedStageBytes / (2 * kTileBytes);
  alignas(1024) uint8_t k[kStages][kTileBytes];
  uint8_t v[kStages][kTileBytes];
  float merge[2][16][D];
  float2 ml[4][16];
  uint64_t full[kStages], empty[kStages];
  uint32_t valid[kStages];  // a bit per 16 keys: the table names a page of the pool
  volatile uint32_t abort_flag;
};

// kWM warps side by side over rows (16 each), 4 / kWM over the keys of a tile.  Compute type: the cache's own 16-bit type, or
// f16 for an E4M3 cache (every E4M3 value is exact in f16; bf16 queries are brought into its range by a power of two per
// row, so they are exact as well down to 2^-38 of the row's largest).
template <int D, typename CacheT, typename QT, int kWM>
__global__ void __launch_bounds__(kPagedThreads, 2) attn_paged_kernel(const PagedParams p, const __grid_constant__ CUtensorMap map_k,
                                                                      const __grid_constant__ CUtensorMap map_v) {
  constexpr bool kE4M3 = std::is_same<CacheT, uint8_t>::value;
  constexpr int kBytes = kE4M3 ? 1 : 2;
  constexpr int kRowBytes = D * kBytes, kBoxBytes = kRowBytes < 128 ? kRowBytes : 128;  // a box: 64 or 128 bytes of a row
  constexpr int kBoxes = kRowBytes / kBoxBytes;
  constexpr int kWK = 4 / kWM, kKeys = kPagedTile / kWK;  // keys of a tile that one warp takes
  using Smem = PagedSmem<D, kBytes>;
  constexpr int kStages = Smem::kStages;
  using Mma = typename std::conditional<kE4M3, TagF16, QT>::type;
  extern __shared__ __align__(1024) uint8_t raw[];
  Smem& s = *reinterpret_cast<Smem*>(raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool aligned = (smem_u32(raw) & 1023u) == 0u;  // the swizzle of the tiles goes by the address
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&s.full[i], 1), mbar_init(&s.empty[i], 4);
    s.abort_flag = 0u;
    fence_barrier_init();
    fence_async_smem();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  __syncthreads();
  pdl_trigger();
  pdl_wait();
  if (!aligned) {
    if (threadIdx.x == 0) p.status[1] = 99u, p.status[0] = 1u;
    return;
  }
  const int64_t total = line_total<false>(p), per_cta = piece_tiles(total, p.own_ctas);
  const int64_t begin = blockIdx.x * per_cta, end = min(total, begin + per_cta);
  if (begin >= end) return;

  if (warp == 4) {  // ---- producer: lane b of a tile's boxes asks for its own part of the pages
    const int box_tokens = min(p.c.page_tokens, kPagedTile), boxes = kPagedTile / box_tokens;
    int stage = 0, issued = 0;
    uint32_t parity = 1u;
    for (int64_t at = begin; at < end;) {
      const PagedUnit u = unit_at<false>(p, at, end);
      const int32_t* row = p.c.table + u.table_slot * p.c.table_stride;
      for (int tile = u.tile; tile < u.tile_end; ++tile, ++at) {
        const int token = tile * kPagedTile + lane * box_tokens;
        const bool wanted = lane < boxes && token < u.key_hi && token + box_tokens > u.key_lo;
        int page = -1;
        if (wanted) page = row[token >> p.c.page_shift];
        const bool load = wanted && page >= 0 && page < p.c.pages;
        const uint32_t loads = __ballot_sync(0xffffffffu, load);
        const bool go = mbar_wait_warp(&s.empty[stage], parity, &s.abort_flag, p.status, 1);
        if (lane == 0) {
          uint32_t valid = 0u;  // per 16 keys
          for (int b = 0; b < boxes; ++b)
            if (loads >> b & 1u) valid |= ((1u << (box_tokens / 16)) - 1u) << (b * (box_tokens / 16));
          s.valid[stage] = valid;
          mbar_expect_tx(&s.full[stage], go ? __popc(loads) * box_tokens * kRowBytes * 2 : 0);
        }
        __syncwarp();
        if (go && load) {
          const uint32_t in_page = (uint32_t)token & (uint32_t)(p.c.page_tokens - 1);
#pragma unroll
          for (int x = 0; x < kBoxes; ++x) {
            const uint32_t off = x * (kPagedTile * kBoxBytes) + lane * box_tokens * kBoxBytes;
            tma_load_5d(smem_u32(s.k[stage]) + off, &map_k, x * (kBoxBytes / kBytes), (int)in_page, u.head, page, p.layer, &s.full[stage]);
            tma_load_5d(smem_u32(s.v[stage]) + off, &map_v, x * (kBoxBytes / kBytes), (int)in_page, u.head, page, p.layer, &s.full[stage]);
          }
        }
        ++issued;
        if (++stage == kStages) stage = 0, parity ^= 1u;
      }
    }
    if (s.abort_flag) {  // copies in flight land before the CTA leaves
      for (int k = max(0, issued - kStages); k < issued; ++k) mbar_wait_teardown(&s.full[k % kStages], (uint32_t)(k / kStages) & 1u);
    }
    return;
  }

  // ---- consumers
  const int wm = warp % kWM, wk = warp / kWM, quad = lane >> 2, c4 = lane & 3;
  int stage = 0;
  uint32_t parity = 0u;
  for (int64_t at = begin; at < end;) {
    const PagedUnit u = unit_at<false>(p, at, end);
    // query rows quad and quad + 8 of this warp's sixteen, as A fragments; row r of them sees keys below `limit`
    uint32_t q[D / 16][4];
    float scale[2];
    int limit[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = wm * 16 + half * 8 + quad;
      const bool there = row < u.rows;
      const PagedRow r = paged_row(p, u, there ? row : 0);
      const uint8_t* src = p.q + 2 * (r.i * p.q_sb + r.h * p.q_sh + r.t * p.q_st);
      limit[half] = u.key_hi - (p.T - 1 - r.t);
      scale[half] = p.scale_log2 * (p.k_scale ? p.k_scale[u.head] : 1.f);
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
            const float2 f = unpack16(q[k][half + x], TagBf16{});
            q[k][half + x] = pack16(f.x * to_f16.a * to_f16.b, f.y * to_f16.a * to_f16.b, TagF16{});
          }
        scale[half] = scale[half] / to_f16.a / to_f16.b;
      }
    }
    float acc[D / 8][4];
#pragma unroll
    for (int j = 0; j < D / 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int tile = u.tile; tile < u.tile_end; ++tile, ++at) {
      mbar_wait_warp(&s.full[stage], parity, &s.abort_flag, p.status, 2);
      const uint32_t kbase = smem_u32(s.k[stage]), vbase = smem_u32(s.v[stage]);
      const int key0 = tile * kPagedTile + wk * kKeys;  // this warp's keys: key0 .. key0 + kKeys
      const uint32_t valid = s.valid[stage] >> (wk * kKeys / 16);
      constexpr uint32_t kAllValid = (1u << (kKeys / 16)) - 1u;
      // not every key of these is there for every row
      const bool special = key0 < u.key_lo || key0 + kKeys > u.key_all || (valid & kAllValid) != kAllValid;
      float sc[kKeys / 8][4];
#pragma unroll
      for (int j = 0; j < kKeys / 8; ++j) {
        sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
        const uint32_t row = wk * kKeys + j * 8 + (lane & 7);
        if constexpr (kE4M3) {
          // a matrix of ldmatrix is 8 keys x 16 codes, four neighbours to a thread: they stand in for k = 2c, 2c+1, 2c+8, 2c+9 of
          // the fragment, and the query fragments above hold the same four neighbours there
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
            ldmatrix4(b, kbase + (col >> 7) * (kPagedTile * 128) + swizzled_offset(row, col & 127u, 128));
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
        if constexpr (kE4M3) {
#pragma unroll
          for (int x = 0; x < D / 32; ++x) {  // matrices: keys 0-7 and 8-15 of 16 codes, then of the next 16
            uint32_t b[4];
            ldmatrix4_trans(b, vbase + swizzled_offset(wk * kKeys + kk * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), x * 32 + (lane >> 4) * 16, kBoxBytes));
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
            ldmatrix4_trans(b, vbase + (col >> 7) * (kPagedTile * 128) +
                                   swizzled_offset(wk * kKeys + kk * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), col & 127u, 128));
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
          const uint32_t row = wk * kKeys + kk;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            float2 f;
            if constexpr (kE4M3) {  // accumulators 2x and 2x + 1: d = 16 x + 4 c + {0, 2} and {1, 3}
              const uint32_t four = *reinterpret_cast<const uint32_t*>(s.v[stage] + swizzled_offset(row, (j >> 1) * 16 + c4 * 4, kBoxBytes));
              f = unpack16(e4m3x2_to_f16x2(__byte_perm(four, 0, j & 1 ? 0x4431 : 0x4420)), TagF16{});
            } else {
              const uint32_t col = j * 16 + c4 * 4;
              f = unpack16(*reinterpret_cast<const uint32_t*>(s.v[stage] + (col >> 7) * (kPagedTile * 128) + swizzled_offset(row, col & 127u, 128)), Mma{});
            }
            if (see0) acc[j][0] = fmaf(p0, f.x, acc[j][0]), acc[j][1] = fmaf(p0, f.y, acc[j][1]);
            if (see1) acc[j][2] = fmaf(p1, f.x, acc[j][2]), acc[j][3] = fmaf(p1, f.y, acc[j][3]);
          }
        }
      }
      mbar_arrive_warp(&s.empty[stage]);
      if (++stage == kStages) stage = 0, parity ^= 1u;
    }

    // ---- the unit's share of this CTA: warps over keys meet, then rows and statistics go to the slot
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    if constexpr (kWK > 1) {
      if (c4 == 0) s.ml[warp][quad] = make_float2(m[0], l[0]), s.ml[warp][quad + 8] = make_float2(m[1], l[1]);
      asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWK; ++w) top = fmaxf(top, s.ml[w * kWM + wm][quad + 8 * h].x);
        const float f = m[h] == -INFINITY ? 0.f : paged_ex2(m[h] - top);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWK; ++w) {
          const float2 x = s.ml[w * kWM + wm][quad + 8 * h];
          sum += x.y * (x.x == -INFINITY ? 0.f : paged_ex2(x.x - top));
        }
        m[h] = top, l[h] = sum;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) acc[j][2 * h] *= f, acc[j][2 * h + 1] *= f;
      }
      // the upper half of the warps hands its sums to the lower half, until one row of warps is left
#pragma unroll
      for (int half = kWK / 2; half >= 1; half /= 2) {
        const bool gives = wk >= half && wk < 2 * half;
        float* buf = &s.merge[kWK == 4 ? (wk & (half - 1)) : wm][0][0];
        if (kWK == 4 && half == 1) buf = &s.merge[1][0][0];  // warp 1 reads and then writes there, warp 0 still reads the other
        if (gives) {
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            *reinterpret_cast<float2*>(buf + quad * D + j * 8 + c4 * 2) = make_float2(acc[j][0], acc[j][1]);
            *reinterpret_cast<float2*>(buf + (quad + 8) * D + j * 8 + c4 * 2) = make_float2(acc[j][2], acc[j][3]);
          }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (wk < half) {
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            const float2 x = *reinterpret_cast<const float2*>(buf + quad * D + j * 8 + c4 * 2);
            const float2 y = *reinterpret_cast<const float2*>(buf + (quad + 8) * D + j * 8 + c4 * 2);
            acc[j][0] += x.x, acc[j][1] += x.y, acc[j][2] += y.x, acc[j][3] += y.y;
          }
        }
      }
    }
    if (wk == 0) {
      const int64_t slot = (int64_t)u.index + blockIdx.x;
      float* out = p.own_acc + slot * p.own_rows * D;
      float2* ml = p.own_ml + slot * p.own_rows;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = wm * 16 + h * 8 + quad;
        if (row >= u.rows) continue;
        if (c4 == 0) ml[row] = make_float2(m[h], l[h]);
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
  }
}

// ---- join -------------------------------------------------------------------------------------------------------------
// One warp per output row.  The pieces' statistics come to the lanes at once, so that what is left to wait for is one
// round of loads: a lane holds D / 32 neighbours of eight pieces at a time.
template <int D, typename QT>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedParams p) {
  constexpr int kPer = D / 32;
  pdl_trigger();
  pdl_wait();
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (w >= (int64_t)p.n * p.Hq * p.T) return;
  const int t = (int)(w % p.T), h = (int)(w / p.T % p.Hq), i = (int)(w / p.T / p.Hq);
  const int g = p.plan.group[i];
  if (g < 0) return;  // behind the last group: left as it was
  const int head = h / p.G, r = t * p.G + h % p.G, len = p.plan.len[i];
  float acc[kPer], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
  if (len - (p.T - 1 - t) > 0) {
    const int first = own_first_key(p, i), tiles = own_tiles(first, len);
    // rows of the row's pieces: piece k of the prefix, then of the own keys, `rows` apart
    int n_prefix = 0, prefix_row = 0;
    int64_t prefix_slot = 0;
    if (first > 0) {
      const int64_t per_cta = piece_tiles(line_total<true>(p), p.prefix_ctas);
      const int lo = max(p.offsets[g], 0), hi = min(p.offsets[g + 1], p.n);
      const int row = (i - lo) * p.R + r, blocks = ceil_div((hi - lo) * p.R, p.prefix_rows);
      const int which = head * blocks + row / p.prefix_rows, ptiles = ceil_div(first, p.prefix_tile);
      const int64_t from = p.plan.g_cum[g] + (int64_t)which * ptiles, cta = from / per_cta;
      n_prefix = (int)((from + ptiles - 1) / per_cta - cta) + 1;
      prefix_slot = p.plan.g_unit[g] + which + cta;
      prefix_row = row % p.prefix_rows;
    }
    const int per = p.c.heads * p.own_blocks, which = head * p.own_blocks + r / p.own_rows;
    const int64_t per_cta = piece_tiles(line_total<false>(p), p.own_ctas), from = (int64_t)p.plan.own_cum[i] * per + (int64_t)which * tiles;
    const int64_t cta = from / per_cta, own_slot = (int64_t)i * per + which + cta;
    const int n_own = (int)((from + tiles - 1) / per_cta - cta) + 1, own_row = r % p.own_rows;
    for (int base = 0; base < n_prefix + n_own; base += 32) {
      const int k = base + lane;
      const bool is_prefix = k < n_prefix;
      const int64_t row = is_prefix ? (prefix_slot + k) * p.prefix_rows + prefix_row : (own_slot + (k - n_prefix)) * p.own_rows + own_row;
      float2 x = make_float2(-INFINITY, 0.f);
      if (k < n_prefix + n_own) x = is_prefix ? p.prefix_ml[row] : p.own_ml[row];
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
      const int count = min(32, n_prefix + n_own - base);
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
  }
  const float inv = l == 0.f ? 0.f : (p.v_scale ? p.v_scale[head] : 1.f) / l;  // a row that sees nothing: zeros, -inf
  uint8_t* out = p.o + 2 * (i * p.o_sb + h * p.o_sh + t * p.o_st + lane * kPer);
  if constexpr (kPer == 4) *reinterpret_cast<uint2*>(out) = make_uint2(pack16(acc[0] * inv, acc[1] * inv, QT{}), pack16(acc[2] * inv, acc[3] * inv, QT{}));
  else *reinterpret_cast<uint32_t*>(out) = pack16(acc[0] * inv, acc[1] * inv, QT{});
  if (lane == 0) p.lse[((int64_t)i * p.Hq + h) * p.T + t] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

}  // namespace fa4b

// ---- host -------------------------------------------------------------------------------------------------------------
namespace fa4b {

template <int D, typename CacheT, typename QT, int kWM>
static int launch_units(const PagedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, int ctas, cudaStream_t st) {
  auto kernel = attn_paged_kernel<D, CacheT, QT, kWM>;
  constexpr int smem = (int)sizeof(PagedSmem<D, std::is_same<CacheT, uint8_t>::value ? 1 : 2>);
  static_assert(smem <= 113 * 1024, "two CTAs per SM");
  FA4B_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  FA4B_CUDA(launch_overlapped(kernel, ctas, kPagedThreads, smem, st, p, mk, mv));
  return FA4B_OK;
}

template <int D, typename CacheT, typename QT>
static int launch_paged(const PagedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  FA4B_CUDA(launch_overlapped(paged_plan_kernel, 1, 1024, 12 * (size_t)p.groups, st, p));
  if (p.groups > 0)
    if (int s = launch_prefix(p, D, std::is_same<CacheT, uint8_t>::value, std::is_same<QT, TagF16>::value, mk, mv, st)) return s;
  const int s = p.own_rows == 16   ? launch_units<D, CacheT, QT, 1>(p, mk, mv, p.own_ctas, st)
                : p.own_rows == 32 ? launch_units<D, CacheT, QT, 2>(p, mk, mv, p.own_ctas, st)
                                   : launch_units<D, CacheT, QT, 4>(p, mk, mv, p.own_ctas, st);
  if (s) return s;
  const int64_t rows = (int64_t)p.n * p.Hq * p.T;
  FA4B_CUDA(launch_overlapped(paged_join_kernel<D, QT>, (unsigned)((rows + 7) / 8), 256, 0, st, p));
  return FA4B_OK;
}

static bool off16(const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) != 0; }

// checks a call and lays its workspace out; `ws` may be NULL (a size query)
static int paged_params(const fa4b_kv_cache* c, const fa4b_attn_paged_args* a, PagedParams* out, size_t* bytes) {
  PagedParams p{};
  if (int s = kv_view(c, &p.c)) return s;
  FA4B_REQUIRE(a != nullptr, FA4B_BAD_ARG, "args is NULL");
  FA4B_REQUIRE(a->n >= 0 && a->n <= kPagedMaxRows, FA4B_BAD_SHAPE, "n=%d: batches of 0 to %d rows are built", a->n, kPagedMaxRows);
  FA4B_REQUIRE(a->T >= 1 && a->T <= kPagedMaxT, FA4B_BAD_SHAPE, "T=%d: 1 to %d query tokens per sequence are built", a->T, kPagedMaxT);
  FA4B_REQUIRE(a->Hq > 0 && a->Hq % c->Hkv == 0, FA4B_BAD_SHAPE, "Hq=%d must be a multiple of Hkv=%d", a->Hq, c->Hkv);
  FA4B_REQUIRE(a->Hq / c->Hkv <= 128, FA4B_BAD_SHAPE, "%d query heads per kv head: at most 128 are built", a->Hq / c->Hkv);
  FA4B_REQUIRE(a->layer >= 0 && a->layer < c->layers, FA4B_BAD_SHAPE, "layer %d of %d", a->layer, c->layers);
  FA4B_REQUIRE(a->q_dtype == FA4B_KV_BF16 || a->q_dtype == FA4B_KV_F16, FA4B_UNSUPPORTED, "queries are bf16 or f16");
  FA4B_REQUIRE(c->dtype == FA4B_KV_E4M3 || a->q_dtype == c->dtype, FA4B_UNSUPPORTED, "a 16-bit cache takes queries of its own type");
  FA4B_REQUIRE(a->groups >= 0 && a->groups <= std::max(a->n, 1), FA4B_BAD_SHAPE, "groups=%d: at most one for each of %d rows", a->groups, a->n);
  FA4B_REQUIRE(a->groups == 0 || (a->group_offsets && a->shared_lens), FA4B_BAD_ARG, "groups need group_offsets and shared_lens");
  FA4B_REQUIRE(a->seqs || a->n <= c->max_seqs, FA4B_BAD_SHAPE, "n=%d rows without a list of slots, and %d slots", a->n, c->max_seqs);
  p.layer = a->layer, p.n = a->n, p.T = a->T, p.Hq = a->Hq, p.G = a->Hq / c->Hkv, p.R = p.T * p.G, p.groups = a->groups;
  p.seqs = a->seqs, p.offsets = a->group_offsets, p.shared = a->shared_lens;
  p.q = static_cast<const uint8_t*>(a->q), p.q_sb = a->q_strides.batch, p.q_sh = a->q_strides.head, p.q_st = a->q_strides.seq;
  p.o = static_cast<uint8_t*>(a->o), p.o_sb = a->o_strides.batch, p.o_sh = a->o_strides.head, p.o_st = a->o_strides.seq;
  p.lse = a->lse;
  for (int64_t s : {p.q_sb, p.q_sh, p.q_st, p.o_sb, p.o_sh, p.o_st})
    FA4B_REQUIRE(s % 8 == 0, FA4B_BAD_ALIGN, "strides of q and o must be multiples of 8 elements");
  FA4B_REQUIRE(!off16(p.q) && !off16(p.o), FA4B_BAD_ALIGN, "q and o must be 16-byte aligned");
  p.scale_log2 = (a->softmax_scale > 0.f ? a->softmax_scale : 1.0f / sqrtf((float)c->D)) * kLog2e;
  if (c->dtype == FA4B_KV_E4M3) p.k_scale = c->k_scale + (int64_t)a->layer * c->Hkv, p.v_scale = c->v_scale + (int64_t)a->layer * c->Hkv;
  const int n_sm = sm_count() > 0 ? sm_count() : 148;
  p.own_rows = p.R <= 16 ? 16 : p.R <= 32 ? 32 : 64;
  p.own_blocks = (p.R + p.own_rows - 1) / p.own_rows;
  p.own_ctas = 2 * n_sm;
  // two blocks of 128 rows over the same keys where the groups have the rows for it: each tile then comes from memory half
  // as often; otherwise the two halves of a CTA take the keys in turn
  p.prefix_rows = p.groups > 0 && (int64_t)p.n * p.R > 128ll * p.groups ? 256 : 128;
  p.prefix_tile = 128, p.prefix_ctas = n_sm;
  const int64_t row_tiles = ((int64_t)c->table_width * c->page_tokens + kPagedTile - 1) / kPagedTile + 1;
  const int64_t prefix_units = p.groups ? (int64_t)c->Hkv * (((int64_t)p.n * p.R + p.prefix_rows - 1) / p.prefix_rows + p.groups) : 0;
  const int64_t own_slots = (int64_t)p.n * c->Hkv * p.own_blocks + p.own_ctas, prefix_slots = p.groups ? prefix_units + p.prefix_ctas : 0;
  // positions on the two lines are counted in 32 bits
  FA4B_REQUIRE(p.n * row_tiles < INT32_MAX && prefix_units * row_tiles < INT32_MAX && own_slots < INT32_MAX, FA4B_BAD_SHAPE,
               "%d rows over tables of %d pages of %d tokens are too many for one call", p.n, c->table_width, c->page_tokens);
  size_t off = 0;
  uint8_t* ws = static_cast<uint8_t*>(a->ws);
  auto take = [&](size_t size) {
    uint8_t* at = ws ? ws + off : nullptr;
    off = align_up(off + size, 256);
    return at;
  };
  const size_t n = p.n, g = p.groups;
  p.plan.slot = reinterpret_cast<int*>(take(4 * n));
  p.plan.len = reinterpret_cast<int*>(take(4 * n));
  p.plan.group = reinterpret_cast<int*>(take(4 * n));
  p.plan.own_cum = reinterpret_cast<int*>(take(4 * (n + 1)));
  p.plan.g_first = reinterpret_cast<int*>(take(4 * g));
  p.plan.g_shared = reinterpret_cast<int*>(take(4 * g));
  p.plan.g_cum = reinterpret_cast<int*>(take(4 * (g + 1)));
  p.plan.g_unit = reinterpret_cast<int*>(take(4 * (g + 1)));
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
  FA4B_REQUIRE((reinterpret_cast<uintptr_t>(a->ws) & 255) == 0, FA4B_BAD_ALIGN, "ws must be 256-byte aligned");
  const bool e4m3 = c->dtype == FA4B_KV_E4M3;
  CUtensorMap mk, mv;
  const uint32_t box = c->D * (e4m3 ? 1 : 2) < 128 ? c->D : 128 / (e4m3 ? 1 : 2);
  const int esz = e4m3 ? 1 : 2;
  const uint64_t dims[5] = {(uint64_t)c->D, (uint64_t)c->page_tokens, (uint64_t)c->Hkv, (uint64_t)c->num_pages, (uint64_t)c->layers};
  const uint32_t boxes[5] = {box, (uint32_t)std::min(c->page_tokens, kPagedTile), 1, 1, 1};
  const uint64_t sk[4] = {(uint64_t)p.c.row_bytes, (uint64_t)p.c.row_bytes * c->page_tokens, (uint64_t)p.c.k_page, (uint64_t)p.c.k_layer};
  const uint64_t sv[4] = {sk[0], sk[1], (uint64_t)p.c.v_page, (uint64_t)p.c.v_layer};
  if (int s = make_tensor_map_5d(&mk, c->k, esz, dims, sk, boxes)) return s;
  if (int s = make_tensor_map_5d(&mv, c->v, esz, dims, sv, boxes)) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool q16 = a->q_dtype == FA4B_KV_F16;
  if (c->D == 128) {
    if (e4m3) return q16 ? launch_paged<128, uint8_t, TagF16>(p, mk, mv, st) : launch_paged<128, uint8_t, TagBf16>(p, mk, mv, st);
    return q16 ? launch_paged<128, uint16_t, TagF16>(p, mk, mv, st) : launch_paged<128, uint16_t, TagBf16>(p, mk, mv, st);
  }
  if (e4m3) return q16 ? launch_paged<64, uint8_t, TagF16>(p, mk, mv, st) : launch_paged<64, uint8_t, TagBf16>(p, mk, mv, st);
  return q16 ? launch_paged<64, uint16_t, TagF16>(p, mk, mv, st) : launch_paged<64, uint16_t, TagBf16>(p, mk, mv, st);
}

}  // extern "C"
