// The prefix units of attention over a paged cache: up to 256 query rows of a group against the keys that its members
// share.  Here a key serves enough rows for the tensor core to be the bound: S = Q K^T and O += P V run on tcgen05 (kind
// f16, M = 128, tiles of 128 keys), S and O live in TMEM, P goes back over S as 16-bit and is the A operand of the
// second product from there.
//
// One CTA per SM.  Warps 0-3 and 4-7: softmax, one thread per row, no exchange between threads (kWide: rows 0-127 and
// 128-255 of the unit, both over every tile; else the same 128 rows, even and odd tiles, joined in TMEM at the end).  While
// one half exponentiates, the tensor core works for the other.  Warp 8 asks for pages by TMA, warp 9 issues the
// products.  An E4M3 cache arrives as codes; warps 10-13 turn each tile into f16 (exact) in the operand ring.
//
// A shared part ends on a multiple of 16 keys (the plan sees to it): the last tile's products take N = its keys and K = its
// keys, so nothing behind them is read and no row needs a mask.
//
// TMEM columns: S 0 and 128, O 256 and 384.
#include "attn_paged.cuh"

#include <type_traits>

namespace fa4b {

constexpr int kPrefixTile = 128;

__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d_tmem), "l"(adesc),
               "l"(bdesc), "r"(idesc), "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d_tmem), "r"(a_tmem),
               "l"(bdesc), "r"(idesc), "r"(accumulate)
               : "memory");
}
// kind::f16: both operands f16 (format 0) or both bf16 (1), f32 accumulators; b_mn: B is MN-major
__device__ __host__ constexpr uint32_t idesc_f16(uint32_t N, uint32_t bf16, uint32_t b_mn) { return idesc_f8(128, N, bf16, bf16, 0, b_mn); }

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
               "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}

template <int D, bool kE4M3, bool kWide>
struct PrefixSmem {
  static constexpr int kSub = 128 * 128;                 // 128 rows of 64 values
  static constexpr int kTile = D / 64 * kSub;            // K or V of 128 keys, or 128 query rows
  static constexpr int kRawTile = 128 * D;
  // without E4M3 tiles to turn, a narrow CTA leaves room for one of the own units beside it
  static constexpr int kRoom = (kWide || kE4M3 ? 224 : 128) * 1024 - (kWide ? 2 : 1) * kTile;
  static constexpr int kRaw = kE4M3 ? 4 : 0;
  static constexpr int kRing = (kRoom - kRaw * kRawTile) / kTile > 8 ? 8 : (kRoom - kRaw * kRawTile) / kTile;
  alignas(1024) uint8_t q[kWide ? 2 : 1][kTile];
  uint8_t ring[kRing][kTile];
  uint8_t raw[kRaw ? kRaw : 1][kRaw ? kRawTile : 16];
  float2 ml[kWide ? 1 : 128];
  uint64_t q_full, q_free, full[kRing], empty[kRing], raw_full[kRaw ? kRaw : 1], raw_empty[kRaw ? kRaw : 1], s_full[2], p_ready[2], o_done[2], drained;
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};

// Where K and V of tile t of a piece of nt tiles stand in the order of loads, which is the order of use: kWide
// K0 V0 K1 V1 ..., else (two tiles under way) K0 K1 V0 K2 V1 K3 ... .
template <bool kWide>
__device__ __forceinline__ int k_at(int t) {
  return kWide ? 2 * t : (t == 0 ? 0 : 2 * t - 1);
}
template <bool kWide>
__device__ __forceinline__ int v_at(int t, int nt) {
  return kWide ? 2 * t + 1 : (t == nt - 1 ? 2 * nt - 1 : 2 * t + 2);
}

// Threads of a CTA: eight warps of softmax, one for pages, one for products, four that turn E4M3 codes.  A narrow 16-bit CTA
// is held to 96 registers (the bound of 576 threads), so that a CTA of own units with up to 224 fits beside it in
// each quarter of the SM (3 x 96 + 224 = 512).
__host__ __device__ constexpr int prefix_threads(bool e4m3) { return e4m3 ? 448 : 320; }
__host__ __device__ constexpr int prefix_bound(bool e4m3, bool wide) { return e4m3 || wide ? prefix_threads(e4m3) : 576; }

// The accumulator of a row scaled where it lies, behind the product that last added to it.
template <int D, typename Smem>
__device__ __forceinline__ void rescale_o(uint32_t to, float f, Smem& s, int w, int steps, uint32_t* status) {
  mbar_wait_warp(&s.o_done[w], (uint32_t)(steps - 1) & 1u, &s.abort_flag, status, 19);
  tc_fence_after();
#pragma unroll 1
  for (int c = 0; c < D; c += 32) {
    uint32_t o[32];
    tmem_ld32(to + c, o);
    tmem_ld_wait(o);
#pragma unroll
    for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
    tmem_st32(to + c, o);
  }
  tmem_st_wait();
}

// A tile of 128 keys that are all there.  Two passes over the scores in TMEM, 32 columns at a time, the next 32 on their way
// while these are worked on (all 128 in registers at once do not fit beside the rest of the row's state).
template <int D, typename Mma, typename Smem>
__device__ __forceinline__ void softmax_tile(uint32_t ts, uint32_t to, float scale, float& m, float& l, bool first, Smem& s, int w, int steps,
                                             uint32_t* status) {
  uint32_t a[2][32];
  tmem_ld32(ts, a[0]);
  float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    tmem_ld_wait(a[c & 1]);
    tmem_ld32(ts + ((c + 1) & 3) * 32, a[(c + 1) & 1]);  // the last one: the first of the second pass
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      t0 = max3(t0, __uint_as_float(a[c & 1][j]), __uint_as_float(a[c & 1][j + 1]));
      t1 = max3(t1, __uint_as_float(a[c & 1][j + 2]), __uint_as_float(a[c & 1][j + 3]));
    }
  }
  const float top = fmaxf(t0, t1) * scale;
  if (__any_sync(0xffffffffu, top > m + 8.f)) {
    const float next = fmaxf(m, top), f = next == -INFINITY ? 1.f : paged_ex2(m - next);
    m = next;
    l *= f;
    if (!first) rescale_o<D>(to, f, s, w, steps, status);
  }
  const float shift = m == -INFINITY ? 0.f : -m;
  const uint64_t scale2 = pack2(scale, scale), shift2 = pack2(shift, shift);
  uint64_t sum0 = pack2(0.f, 0.f), sum1 = sum0;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t out[16];
    tmem_ld_wait(a[c & 1]);
    if (c < 3) tmem_ld32(ts + (c + 1) * 32, a[(c + 1) & 1]);
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      float e0, e1;
      unpack2(fma2(pack2u(a[c & 1][j], a[c & 1][j + 1]), scale2, shift2), e0, e1);
      e0 = paged_ex2(e0), e1 = paged_ex2(e1);
      if (j & 2) sum1 = add2(sum1, pack2(e0, e1)); else sum0 = add2(sum0, pack2(e0, e1));
      out[j / 2] = pack16(e0, e1, Mma{});
    }
    tmem_st16(ts + c * 16, out);  // over scores that have been read: chunk c lies at or below column 16 (c + 1)
  }
  tmem_st_wait();
  float s0, s1;
  unpack2(add2(sum0, sum1), s0, s1);
  l += s0 + s1;
}

template <int D, bool kE4M3, typename QT, bool kWide>
__global__ void __launch_bounds__(prefix_bound(kE4M3, kWide), 1) attn_prefix_kernel(const PagedParams p, const __grid_constant__ CUtensorMap map_k,
                                                                           const __grid_constant__ CUtensorMap map_v) {
  using Smem = PrefixSmem<D, kE4M3, kWide>;
  using Mma = typename std::conditional<kE4M3, TagF16, QT>::type;
  constexpr int kRing = Smem::kRing, kRaw = kE4M3 ? Smem::kRaw : 1, kSub = Smem::kSub;
  constexpr uint32_t kColO = 256;
  constexpr uint32_t kIsBf16 = std::is_same<Mma, TagBf16>::value ? 1 : 0;
  extern __shared__ __align__(1024) uint8_t prefix_raw[];
  Smem& s = *reinterpret_cast<Smem*>(prefix_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool aligned = (smem_u32(prefix_raw) & 1023u) == 0u;
  if (warp == 9) tmem_alloc(&s.tmem_base, 512);
  if (threadIdx.x == 0) {
    mbar_init(&s.q_full, kWide ? 8 : 4);
    mbar_init(&s.q_free, 1);
    for (int i = 0; i < kRing; ++i) mbar_init(&s.full[i], kE4M3 ? 4 : 1), mbar_init(&s.empty[i], 1);
    for (int i = 0; i < kRaw; ++i) mbar_init(&s.raw_full[i], 1), mbar_init(&s.raw_empty[i], 4);
    for (int i = 0; i < 2; ++i) mbar_init(&s.s_full[i], 1), mbar_init(&s.p_ready[i], 4), mbar_init(&s.o_done[i], 1);
    mbar_init(&s.drained, 1);
    s.abort_flag = 0u;
    fence_barrier_init();
    fence_async_smem();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  pdl_wait();
  pdl_trigger();
  PagedWalk<true> walk;
  walk.start(p, blockIdx.x);
  if (!aligned) walk.left = 0;
  if (!aligned && threadIdx.x == 0) p.status[1] = 98u, p.status[0] = 1u;

  if (warp == 8) {  // ---- pages
    const int box_tokens = min(p.c.page_tokens, kPagedBox), boxes = kPrefixTile / box_tokens;
    constexpr int kBytes = kE4M3 ? 1 : 2, kBoxBytes = D * kBytes < 128 ? D * kBytes : 128, kBoxes = D * kBytes / kBoxBytes;
    constexpr int kSlots = kE4M3 ? kRaw : kRing;
    uint64_t* full = kE4M3 ? s.raw_full : s.full;
    uint64_t* empty = kE4M3 ? s.raw_empty : s.empty;
    int slot = 0, issued = 0;
    uint32_t parity = 1u;
    while (!walk.done()) {
      const PagedUnit u = walk.next(p);
      const int32_t* row = p.c.table + u.table_slot * p.c.table_stride;
      const int nt = u.tile_end - u.tile;
      if (nt == 0) continue;
      for (int x = 0; x < 2 * nt; ++x) {
        bool is_v;
        int t;
        if constexpr (kWide) is_v = x & 1, t = x >> 1;
        else if (x == 2 * nt - 1) is_v = true, t = nt - 1;
        else if (x == 0) is_v = false, t = 0;
        else is_v = !(x & 1), t = is_v ? x / 2 - 1 : (x + 1) / 2;
        const int token = (u.tile + t) * kPrefixTile + lane * box_tokens;
        const bool load = lane < boxes && token < u.key_hi;
        const int page = load ? row[token >> p.c.page_shift] : 0;  // the plan has looked at these entries
        const int n_loads = __popc(__ballot_sync(0xffffffffu, load));
        const bool go = mbar_wait_warp(&empty[slot], parity, &s.abort_flag, p.status, 11);
        if (lane == 0) mbar_expect_tx(&full[slot], go ? n_loads * box_tokens * D * kBytes : 0);
        __syncwarp();
        if (go && load) {
          const uint32_t in_page = (uint32_t)token & (uint32_t)(p.c.page_tokens - 1);
          const uint32_t dst = kE4M3 ? smem_u32(s.raw[slot]) : smem_u32(s.ring[slot]);
#pragma unroll
          for (int b = 0; b < kBoxes; ++b)
            tma_load_5d(dst + b * (128 * kBoxBytes) + lane * box_tokens * kBoxBytes, is_v ? &map_v : &map_k, b * (kBoxBytes / kBytes), (int)in_page,
                        u.head, page, p.layer, &full[slot]);
        }
        ++issued;
        if (++slot == kSlots) slot = 0, parity ^= 1u;
      }
    }
    if (s.abort_flag)  // copies in flight land before the CTA leaves
      for (int k = max(0, issued - kSlots); k < issued; ++k) mbar_wait_teardown(&full[k % kSlots], (uint32_t)(k / kSlots) & 1u);
  } else if (warp == 9) {  // ---- products
    if (lane == 0) {
      int base = 0, units = 0, steps[2] = {0, 0};
      bool ok = true;
      auto wait_full = [&](int x) { ok = mbar_wait(&s.full[(base + x) % kRing], (uint32_t)((base + x) / kRing) & 1u, &s.abort_flag, p.status, 12) && ok; };
      while (!walk.done()) {
        const PagedUnit u = walk.next(p);
        const int nt = u.tile_end - u.tile;
        if (nt == 0) continue;
        const int halves = kWide ? (u.rows > 128 ? 2 : 1) : (nt > 1 ? 2 : 1);
        auto keys_of = [&](int t) { return min(kPrefixTile, u.key_hi - (u.tile + t) * kPrefixTile); };
        auto scores = [&](int w, int t) {  // S of half w = Q . K(t)
          if (ok) {
            const uint32_t idesc = idesc_f16(keys_of(t), kIsBf16, 0), qa = smem_u32(s.q[kWide ? w : 0]), ka = smem_u32(s.ring[(base + k_at<kWide>(t)) % kRing]);
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              mma_f16_ss(tmem + w * 128, make_tile_desc(qa + (k >> 2) * kSub + (k & 3) * 32, 128), make_tile_desc(ka + (k >> 2) * kSub + (k & 3) * 32, 128), idesc, k > 0);
          }
          mma_commit(&s.s_full[w]);
        };
        auto values = [&](int w, int t, bool first) {  // O of half w += P . V(t)
          ok = mbar_wait(&s.p_ready[w], (uint32_t)steps[w] & 1u, &s.abort_flag, p.status, 13) && ok;
          ++steps[w];
          tc_fence_after();
          if (ok) {
            const uint32_t idesc = idesc_f16(D, kIsBf16, 1), va = smem_u32(s.ring[(base + v_at<kWide>(t, nt)) % kRing]);
            const int ks = keys_of(t) / 16;
            for (int k = 0; k < ks; ++k)
              mma_f16_ts(tmem + kColO + w * 128, tmem + w * 128 + k * 8, make_sdesc(va + k * 2048, kSub, 1024, kSwz128), idesc, !(first && k == 0));
          }
          mma_commit(&s.o_done[w]);
        };
        auto release = [&](int x) { mma_commit(&s.empty[(base + x) % kRing]); };
        ok = mbar_wait(&s.q_full, (uint32_t)units & 1u, &s.abort_flag, p.status, 14) && ok;
        ++units;
        if constexpr (kWide) {
          wait_full(0);
          for (int w = 0; w < halves; ++w) scores(w, 0);
          release(0);
          for (int t = 0; t < nt; ++t) {
            wait_full(v_at<true>(t, nt));
            if (t + 1 < nt) wait_full(k_at<true>(t + 1));
            for (int w = 0; w < halves; ++w) {
              values(w, t, t == 0);
              if (t + 1 < nt) scores(w, t + 1);
            }
            release(v_at<true>(t, nt));
            if (t + 1 < nt) release(k_at<true>(t + 1));
            if (t == max(nt - 2, 0)) mma_commit(&s.q_free);  // the last scores of the unit have been issued
          }
        } else {
          for (int t = 0; t < halves; ++t) {
            wait_full(k_at<false>(t));
            scores(t, t);
            release(k_at<false>(t));
          }
          if (nt <= 2) mma_commit(&s.q_free);
          for (int t = 0; t < nt; ++t) {
            wait_full(v_at<false>(t, nt));
            values(t & 1, t, t < 2);
            release(v_at<false>(t, nt));
            if (t + 2 < nt) {
              wait_full(k_at<false>(t + 2));
              scores(t & 1, t + 2);
              release(k_at<false>(t + 2));
              if (t + 3 == nt) mma_commit(&s.q_free);
            }
          }
        }
        base += 2 * nt;
      }
      mma_commit(&s.drained);
      mbar_wait_teardown(&s.drained, 0u);
    }
    __syncwarp();
  } else if (kE4M3 && warp >= 10) {  // ---- codes to f16
    const int w = warp - 10, tid = w * 32 + lane;
    constexpr int kChunks = D / 16, kRawRow = D;  // 16 codes each
    int n = 0;
    while (!walk.done()) {
      const PagedUnit u = walk.next(p);
      const int nt = u.tile_end - u.tile;
      if (nt == 0) continue;
      for (int x = 0; x < 2 * nt; ++x, ++n) {
        const int raw = n % kRaw, slot = n % kRing;
        mbar_wait_warp(&s.raw_full[raw], (uint32_t)(n / kRaw) & 1u, &s.abort_flag, p.status, 15);
        mbar_wait_warp(&s.empty[slot], ((uint32_t)(n / kRing) & 1u) ^ 1u, &s.abort_flag, p.status, 16);
        // eight chunks per thread (four for D = 64), all read before the first is written
        uint4 in[kChunks];
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          const uint32_t at = tid + i * 128;
          in[i] = *reinterpret_cast<const uint4*>(s.raw[raw] + swizzled_offset(at / kChunks, (at % kChunks) * 16, kRawRow));
        }
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          const uint32_t at = tid + i * 128, row = at / kChunks, c = at % kChunks;
          const uint32_t x[4] = {in[i].x, in[i].y, in[i].z, in[i].w};
          uint32_t out[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) out[2 * e] = e4m3x2_to_f16x2(x[e]), out[2 * e + 1] = e4m3x2_to_f16x2(x[e] >> 16);
          uint8_t* sub = s.ring[slot] + (c >> 2) * kSub;
          *reinterpret_cast<uint4*>(sub + swizzled_offset(row, (c & 3) * 32, 128)) = make_uint4(out[0], out[1], out[2], out[3]);
          *reinterpret_cast<uint4*>(sub + swizzled_offset(row, (c & 3) * 32 + 16, 128)) = make_uint4(out[4], out[5], out[6], out[7]);
        }
        fence_async_smem();
        mbar_arrive_warp(&s.full[slot]);
        mbar_arrive_warp(&s.raw_empty[raw]);
      }
    }
  } else if (warp < 8) {  // ---- softmax: thread = row
    const int w = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's quarter of the lanes
    const uint32_t ts = tmem + lanes + w * 128, to = tmem + lanes + kColO + w * 128;
    int units = 0, steps = 0, other_steps = 0;  // tiles that this half, and the other, have done
    while (!walk.done()) {
      const PagedUnit u = walk.next(p);
      const int nt = u.tile_end - u.tile;
      if (nt == 0) continue;
      const int row = (kWide ? w * 128 : 0) + r;
      const bool there = row < u.rows, active = (kWide ? w * 128 : 0) + (warp & 3) * 32 < u.rows;
      const bool half_there = kWide ? w * 128 < u.rows : w < nt;
      if (units > 0) mbar_wait_warp(&s.q_free, (uint32_t)(units - 1) & 1u, &s.abort_flag, p.status, 17);
      float scale = p.scale_log2;
      if (active) {  // the query row, swizzled into shared memory
        const PagedRow pr = paged_row(p, u, there ? row : 0);
        const uint4* src = reinterpret_cast<const uint4*>(p.q + 2 * (pr.i * p.q_sb + pr.h * p.q_sh + pr.t * p.q_st));
        uint4 x[D / 8];
#pragma unroll
        for (int c = 0; c < D / 8; ++c) x[c] = src[c];
        if constexpr (kE4M3) scale = e4m3_query_row<QT, D / 8>(x, scale * p.k_scale[u.head]);
        if (kWide || w == 0) {
#pragma unroll
          for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4*>(s.q[kWide ? w : 0] + (c >> 3) * kSub + swizzled_offset(r, (c & 7) * 16, 128)) = x[c];
        }
      }
      if (kWide || w == 0) {
        fence_async_smem();
        mbar_arrive_warp(&s.q_full);
      }
      ++units;
      float m = -INFINITY, l = 0.f;
      if (half_there)
        for (int t = kWide ? 0 : w; t < nt; t += kWide ? 1 : 2) {
          const int keys = min(kPrefixTile, u.key_hi - (u.tile + t) * kPrefixTile);
          mbar_wait_warp(&s.s_full[w], (uint32_t)steps & 1u, &s.abort_flag, p.status, 18);
          tc_fence_after();
          if (active) {
            if (keys == kPrefixTile) {
              softmax_tile<D, Mma>(ts, to, scale, m, l, t < (kWide ? 1 : 2), s, w, steps, p.status);
              tc_fence_before();
              mbar_arrive_warp(&s.p_ready[w]);
              ++steps;
              continue;
            }
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              if (c * 64 >= keys) break;
              uint32_t a[32], b[32];
              tmem_ld32(ts + c * 64, a);
              tmem_ld32(ts + c * 64 + 32, b);
              tmem_ld_wait(a);
              tmem_ld_wait(b);
              if (keys >= c * 64 + 64) {
                float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                  t0 = max3(t0, __uint_as_float(a[j]), __uint_as_float(a[j + 1]));
                  t1 = max3(t1, __uint_as_float(b[j]), __uint_as_float(b[j + 1]));
                }
                top = max3(top, t0, t1);
              } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                  if (c * 64 + j < keys) top = fmaxf(top, __uint_as_float(a[j]));
                  if (c * 64 + 32 + j < keys) top = fmaxf(top, __uint_as_float(b[j]));
                }
              }
            }
            top *= scale;
            // the reference point moves when it has to (see the own units); the accumulator is then scaled where it lies
            if (__any_sync(0xffffffffu, top > m + 8.f)) {
              const float next = fmaxf(m, top), f = next == -INFINITY ? 1.f : paged_ex2(m - next);
              const bool first = t < (kWide ? 1 : 2);
              m = next;
              l *= f;
              if (!first) rescale_o<D>(to, f, s, w, steps, p.status);
            }
            const float shift = m == -INFINITY ? 0.f : -m;
            const uint64_t scale2 = pack2(scale, scale), shift2 = pack2(shift, shift);
            uint64_t sum2 = pack2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              if (c * 32 >= keys) break;
              uint32_t a[32], out[16];
              tmem_ld32(ts + c * 32, a);
              tmem_ld_wait(a);
              if (keys < c * 32 + 32) {
#pragma unroll
                for (int j = 16; j < 32; ++j) a[j] = 0xff800000u;  // only 16 of these keys are there
              }
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                float e0, e1;
                unpack2(fma2(pack2u(a[j], a[j + 1]), scale2, shift2), e0, e1);
                e0 = paged_ex2(e0), e1 = paged_ex2(e1);
                if (j >= 16 && keys < c * 32 + 32) e0 = e1 = 0.f;
                sum2 = add2(sum2, pack2(e0, e1));
                out[j / 2] = pack16(e0, e1, Mma{});
              }
              tmem_st16(ts + c * 16, out);
            }
            tmem_st_wait();
            float s0, s1;
            unpack2(sum2, s0, s1);
            l += s0 + s1;
          }
          tc_fence_before();
          mbar_arrive_warp(&s.p_ready[w]);
          ++steps;
        }
      // ---- the piece goes to its slot
      const int64_t slot = (int64_t)u.index + blockIdx.x;
      float* out = p.prefix_acc + (slot * p.prefix_rows + row) * D;
      if constexpr (kWide) {
        if (half_there) {
          mbar_wait_warp(&s.o_done[w], (uint32_t)(steps - 1) & 1u, &s.abort_flag, p.status, 20);
          tc_fence_after();
          if (active) {
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_ld32(to + c, o);
              tmem_ld_wait(o);
              if (there)
#pragma unroll
                for (int j = 0; j < 32; j += 8) store8(out + c + j, o + j);
            }
            if (there) p.prefix_ml[slot * p.prefix_rows + row] = make_float2(m, l);
          }
          tc_fence_before();
        }
      } else {
        // both halves hold sums of the same rows: each joins one half of the columns
        other_steps += w == 0 ? nt / 2 : (nt + 1) / 2;
        if (w == 0) s.ml[r] = make_float2(m, l);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        float2 x;
        if (w == 1) x = s.ml[r], s.ml[r] = make_float2(m, l);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (w == 0) x = s.ml[r];
        const bool both = nt > 1;
        if (w < nt) mbar_wait_warp(&s.o_done[w], (uint32_t)(steps - 1) & 1u, &s.abort_flag, p.status, 21);
        if (w != 0 || both) mbar_wait_warp(&s.o_done[w ^ 1], (uint32_t)(other_steps - 1) & 1u, &s.abort_flag, p.status, 22);
        tc_fence_after();
        const float top = fmaxf(m, x.x);
        const float mine = m == -INFINITY ? 0.f : paged_ex2(m - top), theirs = x.x == -INFINITY ? 0.f : paged_ex2(x.x - top);
        if (active) {
          const float f0 = w == 0 ? mine : theirs, f1 = w == 0 ? theirs : mine;
          const uint32_t t0 = tmem + lanes + kColO;
#pragma unroll 1
          for (int c = w * (D / 2); c < (w + 1) * (D / 2); c += 16) {
            uint32_t a[16], b[16];
            tmem_ld16(t0 + c, a);
            if (both) tmem_ld16(t0 + 128 + c, b);
            tmem_ld_wait16(a);
            if (both) tmem_ld_wait16(b);
#pragma unroll
            for (int j = 0; j < 16; ++j) a[j] = __float_as_uint(__uint_as_float(a[j]) * f0 + (both ? __uint_as_float(b[j]) * f1 : 0.f));
            if (there) store8(out + c, a), store8(out + c + 8, a + 8);
          }
          if (there && w == 0) p.prefix_ml[slot * p.prefix_rows + row] = make_float2(top, l * mine + x.y * theirs);
        }
        tc_fence_before();
        asm volatile("bar.sync 1, 256;" ::: "memory");  // O and ml are free for the next unit
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

template <int D, bool kE4M3, typename QT, bool kWide>
static int launch_prefix_of(const PagedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  auto kernel = attn_prefix_kernel<D, kE4M3, QT, kWide>;
  constexpr int smem = (int)sizeof(PrefixSmem<D, kE4M3, kWide>);
  static_assert(smem <= 227 * 1024, "shared memory of one CTA");
  static_assert(PrefixSmem<D, kE4M3, kWide>::kRing >= 3, "two tiles under way and one on its way");
  static std::atomic<uint64_t> allowed{0};
  if (int s = allow_smem(kernel, smem, allowed)) return s;
  FA4B_CUDA(launch_overlapped(kernel, p.prefix_workers, prefix_threads(kE4M3), smem, st, p, mk, mv));
  return FA4B_OK;
}

template <int D, bool kE4M3, typename QT>
static int launch_prefix_wide(const PagedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  return p.prefix_rows == 256 ? launch_prefix_of<D, kE4M3, QT, true>(p, mk, mv, st) : launch_prefix_of<D, kE4M3, QT, false>(p, mk, mv, st);
}

int launch_prefix(const PagedParams& p, int D, bool e4m3, bool q_f16, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  if (D == 128) {
    if (e4m3) return q_f16 ? launch_prefix_wide<128, true, TagF16>(p, mk, mv, st) : launch_prefix_wide<128, true, TagBf16>(p, mk, mv, st);
    return q_f16 ? launch_prefix_wide<128, false, TagF16>(p, mk, mv, st) : launch_prefix_wide<128, false, TagBf16>(p, mk, mv, st);
  }
  if (e4m3) return q_f16 ? launch_prefix_wide<64, true, TagF16>(p, mk, mv, st) : launch_prefix_wide<64, true, TagBf16>(p, mk, mv, st);
  return q_f16 ? launch_prefix_wide<64, false, TagF16>(p, mk, mv, st) : launch_prefix_wide<64, false, TagBf16>(p, mk, mv, st);
}

}  // namespace fa4b
