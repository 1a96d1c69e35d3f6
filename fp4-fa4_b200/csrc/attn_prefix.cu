// The prefix units of attention over a paged cache: up to 256 query rows of a group against the keys that its members
// share.  Here a key serves enough rows for the tensor core to be the bound: S = Q K^T and O += P V run on tcgen05 (kind
// f16, M = 128, tiles of 128 keys), S and O live in TMEM, P goes back over S as 16-bit and is the A operand of the
// second product from there.
//
// One CTA per SM.  Warps 0-3 and 4-7: softmax, one thread per row, no exchange between threads (kWide: rows 0-127 and
// 128-255 of the unit, both over every key; else the same 128 rows, the first and the last 64 keys of a tile, joined in
// TMEM at the end).  Either half works in steps of 64 keys on two score buffers of its own: while it exponentiates one,
// the tensor core fills the other, so that it hardly ever waits (with one buffer of 128 keys per half a step spent as long
// waiting for P V and the next Q K^T as exponentiating).  Warp 8 asks for pages by TMA, warps 9 and 10 issue the products of the
// halves.  An E4M3 cache arrives as codes; warps 11-14 turn each tile into f16 (exact) in the operand ring.
//
// 2048 rows (128 sequences of 4 tokens and 4 query heads) over 32768 keys and 8 kv heads, D 128, bf16: 255 us (275 GFLOP: 0.66 of
// the rate measured for a library's product of large matrices; one buffer 281 us, one issuing warp 482).  The products bound it: one of
// 64 keys takes about 85 cycles, as long as one of 128, because the query operand comes from shared memory for each (TMEM is full),
// so a step of both halves, 16 products of scores and 8 of values, is 1900 of the 2130 cycles that it takes.  Scores of 128
// keys at once would leave no second buffer and were slower (382 against 333 us for the call).  With 128 rows and 8k keys it is 13.5
// us: 7 of them are the beginning (plan, query rows, first pages) and the end (the sums out of TMEM).
//
// A shared part ends on a multiple of 16 keys (the plan sees to it): the last tile's products take N = its keys and K = its
// keys, so nothing behind them is read and no row needs a mask.
//
// TMEM columns: S 0 and 64 of the first half, 128 and 192 of the second (P in the lower 32 of each), O 256 and 384.
#include "attn_paged.cuh"

#include <cstddef>
#include <type_traits>

namespace fa4b {

constexpr int kPrefixTile = kPagedPrefixTile, kStep = 64;

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
  static constexpr int kRoom = 224 * 1024 - (kWide ? 2 : 1) * kTile;
  static constexpr int kRaw = kE4M3 ? 4 : 0;
  static constexpr int kRing = (kRoom - kRaw * kRawTile) / kTile > 8 ? 8 : (kRoom - kRaw * kRawTile) / kTile;
  alignas(1024) uint8_t q[kWide ? 2 : 1][kTile];
  uint8_t ring[kRing][kTile];
  uint8_t raw[kRaw ? kRaw : 1][kRaw ? kRawTile : 16];
  float2 ml[2][kWide ? 1 : 128];
  uint64_t q_full, q_free, full[kRing], empty[kRing], raw_full[kRaw ? kRaw : 1], raw_empty[kRaw ? kRaw : 1], s_full[2][2], p_ready[2][2], o_done[2][2], drained;  // [half][score buffer]
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
  // the struct without what its alignment adds
  static constexpr int kUsed = ((kWide ? 2 : 1) + kRing) * kTile + (kRaw ? kRaw * kRawTile : 16) + (kWide ? 1 : 128) * 16 +
                               8 * (2 + 2 * kRing + 2 * (kRaw ? kRaw : 1) + 13) + 16;
};

// Keys of step `step` of a half of a piece whose keys end at `keys`, counted from its first tile; 0 behind the last.
template <bool kWide>
__device__ __forceinline__ int step_keys(int keys, int half, int step) {
  const int first = kWide ? step * kStep : step * kPrefixTile + half * kStep;
  return max(0, min(kStep, keys - first));
}

// eight warps of softmax, one for pages, two for products, four that turn E4M3 codes
__host__ __device__ constexpr int prefix_threads(bool e4m3) { return e4m3 ? 480 : 352; }

// The accumulator of a row scaled where it lies, behind the product of the step before (`done`, `parity`).  A barrier of its
// own for each score buffer: a step's scores are only there when the product of the step before last is, so that a
// wait is never two phases behind.
template <int D, typename Smem>
__device__ __forceinline__ void rescale_o(uint32_t to, float f, Smem& s, uint64_t* done, uint32_t parity, uint32_t* status) {
  mbar_wait_warp(done, parity, &s.abort_flag, status, 19);
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

// One step of a row: scores out of TMEM, probabilities back in as 16-bit.  keys: 16 to 64 in sixteens; kFull: 64 (with
// the other case in the same code every exponential hangs on a branch).  kLean: 32 scores in registers at a time, read once
// for their maximum and once more to be used (with the threads that turn codes there are 128 registers for each).
template <int D, typename Mma, bool kLean, bool kFull, typename Smem>
__device__ __forceinline__ void softmax_step(uint32_t ts, uint32_t to, int keys, float scale, float& m, float& l, Smem& s, uint64_t* before,
                                             uint32_t parity_before, bool first, uint32_t* status) {
  uint32_t a[kLean ? 1 : 2][32];
  if constexpr (!kLean) {
    tmem_ld32(ts, a[0]);
    tmem_ld32(ts + 32, a[1]);
    tmem_ld_wait(a[0]);
    tmem_ld_wait(a[1]);
  }
  float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t(&x)[32] = a[kLean ? 0 : c];
    if constexpr (kLean) {
      tmem_ld32(ts + c * 32, x);
      tmem_ld_wait(x);
    }
    if constexpr (!kFull) {  // the rest of the buffer is what an earlier step left
#pragma unroll
      for (int j = 0; j < 32; j += 16)
        if (keys <= c * 32 + j)
#pragma unroll
          for (int e = 0; e < 16; ++e) x[j + e] = 0xff800000u;
    }
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      t0 = max3(t0, __uint_as_float(x[j]), __uint_as_float(x[j + 1]));
      t1 = max3(t1, __uint_as_float(x[j + 2]), __uint_as_float(x[j + 3]));
    }
  }
  const float top = fmaxf(t0, t1) * scale;
  // the reference point moves when it has to (see the own units); the accumulator is then scaled where it lies
  if (__any_sync(0xffffffffu, top > m + 8.f)) {
    const float next = fmaxf(m, top), f = next == -INFINITY ? 1.f : paged_ex2(m - next);
    m = next;
    l *= f;
    if (!first) rescale_o<D>(to, f, s, before, parity_before, status);
  }
  const float shift = m == -INFINITY ? 0.f : -m;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t(&x)[32] = a[kLean ? 0 : c];
    if constexpr (kLean) {
      tmem_ld32(ts + c * 32, x);
      tmem_ld_wait(x);
    }
    uint32_t out[16];
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[i] = paged_ex2(fmaf(__uint_as_float(x[j + i]), scale, shift));
        if constexpr (!kFull)
          if (c * 32 + j >= 16 && keys <= (c * 32 + j) / 16 * 16) e[i] = 0.f;  // not there
        sum[i] += e[i];
      }
      out[j / 2] = pack16(e[0], e[1], Mma{}), out[j / 2 + 1] = pack16(e[2], e[3], Mma{});
    }
    tmem_st16(ts + c * 16, out);
  }
  tmem_st_wait();
  l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

template <int D, bool kE4M3, typename QT, bool kWide>
__global__ void __launch_bounds__(prefix_threads(kE4M3), 1) attn_prefix_kernel(const PagedParams p, const __grid_constant__ CUtensorMap map_k,
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
    mbar_init(&s.q_free, 2);
    for (int i = 0; i < kRing; ++i) mbar_init(&s.full[i], kE4M3 ? 4 : 1), mbar_init(&s.empty[i], 2);
    for (int i = 0; i < kRaw; ++i) mbar_init(&s.raw_full[i], 1), mbar_init(&s.raw_empty[i], 4);
    for (int i = 0; i < 2; ++i) {
      for (int j = 0; j < 2; ++j) mbar_init(&s.s_full[i][j], 1), mbar_init(&s.p_ready[i][j], 4), mbar_init(&s.o_done[i][j], 1);
    }
    mbar_init(&s.drained, 2);
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
  walk.start(p, blockIdx.x, {&p.head->prefix, nullptr, p.g_cum});
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
        // the order of use: kWide (a tile is two steps, both score buffers) K0 V0 K1 V1 ..., else (a tile is one step, the
        // buffers hold two tiles) K0 K1 V0 K2 V1 ...
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
  } else if (warp == 9 || warp == 10) {  // ---- products of the first and of the second half
    // The warp walks together and one lane issues: what a product takes (descriptors, columns) is then the same in all lanes and
    // costs an addition each (in a branch of one lane: 60 to 120 cycles an instruction).  One warp for both halves would
    // spend as long between its products as the tensor core on them.
    const int w = warp - 9;
    const bool leader = elect_one();
    const uint64_t q_desc = make_tile_desc(smem_u32(s.q[kWide ? w : 0]), 128), k_desc = make_tile_desc(smem_u32(s.ring[0]), 128),
                   v_desc = make_sdesc(smem_u32(s.ring[0]), kSub, 1024, kSwz128);
    constexpr uint32_t kIdescV = idesc_f16(D, kIsBf16, 1);
    const uint32_t scol = tmem + w * 128, ocol = tmem + kColO + w * 128;
    int slot = 0, units = 0;
    uint32_t parity = 0u, phases = 0u;  // of the ring; of the probabilities that are awaited next, a bit per buffer
    bool ok = true;
    auto take = [&]() {  // the next tile of the ring: tiles are used in the order of their loads
      ok = mbar_wait_warp(&s.full[slot], parity, &s.abort_flag, p.status, 12) && ok;
      const int got = slot;
      if (++slot == kRing) slot = 0, parity ^= 1u;
      return got;
    };
    auto commit = [&](uint64_t* bar) {
      if (leader) mma_commit(bar);
    };
    auto scores = [&](int buf, int n, int tile, int row) {  // S = Q . K, n keys from row `row` of a tile
      const uint32_t idesc = idesc_f16(n, kIsBf16, 0);
      const uint64_t kd = k_desc + tile * (Smem::kTile >> 4) + row * 8;
      if (leader) {
        if (ok)
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_f16_ss(scol + buf * kStep, q_desc + ((k >> 2) * kSub + (k & 3) * 32) / 16, kd + ((k >> 2) * kSub + (k & 3) * 32) / 16, idesc, k > 0);
        mma_commit(&s.s_full[w][buf]);
      }
    };
    auto values = [&](int buf, int n, int tile, int row, bool first) {  // O += P . V
      const uint64_t vd = v_desc + tile * (Smem::kTile >> 4) + row * 8;
      const uint32_t pcol = scol + buf * kStep;
      ok = mbar_wait_warp(&s.p_ready[w][buf], phases >> buf & 1u, &s.abort_flag, p.status, 13) && ok;
      phases ^= 1u << buf;
      tc_fence_after();
      if (leader) {
        if (ok) {
          mma_f16_ts(ocol, pcol, vd, kIdescV, !first);
          if (n == kStep) {
#pragma unroll
            for (int k = 1; k < kStep / 16; ++k) mma_f16_ts(ocol, pcol + k * 8, vd + k * 128, kIdescV, 1);
          } else {
            for (int k = 1; k < n / 16; ++k) mma_f16_ts(ocol, pcol + k * 8, vd + k * 128, kIdescV, 1);
          }
        }
        mma_commit(&s.o_done[w][buf]);
      }
    };
    while (!walk.done()) {
      const PagedUnit u = walk.next(p);
      const int nt = u.tile_end - u.tile;
      if (nt == 0) continue;
      const int piece = kWide && w * 128 >= u.rows ? 0 : min(u.key_hi - u.tile * kPrefixTile, nt * kPrefixTile);  // keys; a half without rows takes none
      ok = mbar_wait_warp(&s.q_full, (uint32_t)units & 1u, &s.abort_flag, p.status, 14) && ok;
      ++units;
      if constexpr (kWide) {
        auto keys = [&](int step) { return min(kStep, piece - step * kStep); };
        int tile = take();
        if (keys(0) > 0) scores(0, keys(0), tile, 0);
        if (keys(1) > 0) scores(1, keys(1), tile, kStep);
        commit(&s.empty[tile]);
        if (nt == 1) commit(&s.q_free);
        for (int t = 0; t < nt; ++t) {
          const int v = take();
          const bool more = t + 1 < nt;
          if (keys(2 * t) > 0) values(0, keys(2 * t), v, 0, t == 0);
          if (more) tile = take();
          if (more && keys(2 * t + 2) > 0) scores(0, keys(2 * t + 2), tile, 0);
          if (keys(2 * t + 1) > 0) values(1, keys(2 * t + 1), v, kStep, false);
          commit(&s.empty[v]);
          if (more) {
            if (keys(2 * t + 3) > 0) scores(1, keys(2 * t + 3), tile, kStep);
            commit(&s.empty[tile]);
            if (t + 2 == nt) commit(&s.q_free);  // the last scores of the unit have been issued
          }
        }
      } else {
        auto keys = [&](int t) { return min(kStep, piece - t * kPrefixTile - w * kStep); };
        for (int t = 0; t < min(nt, 2); ++t) {
          const int tile = take();
          if (keys(t) > 0) scores(t, keys(t), tile, w * kStep);
          commit(&s.empty[tile]);
        }
        if (nt <= 2) commit(&s.q_free);
        for (int t = 0; t < nt; ++t) {
          const int v = take();
          if (keys(t) > 0) values(t & 1, keys(t), v, w * kStep, t == 0);
          commit(&s.empty[v]);
          if (t + 2 < nt) {
            const int tile = take();
            if (keys(t + 2) > 0) scores(t & 1, keys(t + 2), tile, w * kStep);
            commit(&s.empty[tile]);
            if (t + 3 == nt) commit(&s.q_free);
          }
        }
      }
    }
    commit(&s.drained);
    mbar_wait_teardown(&s.drained, 0u);
  } else if (kE4M3 && warp >= 11) {  // ---- codes to f16
    const int w = warp - 11, tid = w * 32 + lane;
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
    int units = 0;
    uint32_t phases = 0u, other_phases = 0u;  // a bit per buffer, of this half and of the other
    while (!walk.done()) {
      const PagedUnit u = walk.next(p);
      const int nt = u.tile_end - u.tile;
      if (nt == 0) continue;
      const bool two = !kWide && prefix_in_two(p, u.rows);
      const int row = kWide ? w * 128 + r : two ? r & 63 : r;
      const bool mine = !two || r >> 6 == w;                          // of this half
      const bool loads = (row & ~31) < u.rows, active = loads && mine, there = row < u.rows && mine;
      const int piece = min(u.key_hi - u.tile * kPrefixTile, nt * kPrefixTile);
      const int n_steps = kWide ? (w * 128 < u.rows ? (piece + kStep - 1) / kStep : 0) : (piece - w * kStep + kPrefixTile - 1) / kPrefixTile;
      if (units > 0) mbar_wait_warp(&s.q_free, (uint32_t)(units - 1) & 1u, &s.abort_flag, p.status, 17);
      float scale = p.scale_log2;
      if (loads) {  // the query row, swizzled into shared memory
        const PagedRow pr = paged_row(p, u, row < u.rows ? row : 0);
        const uint4* src = reinterpret_cast<const uint4*>(p.q + 2 * (pr.i * p.q_sb + pr.h * p.q_sh + pr.t * p.q_st));
        uint8_t* dst = s.q[kWide ? w : 0];
        if constexpr (kE4M3) {  // in f16; the factor's sign moves into the row
          RowShift to_f16{1.f, 1.f};
          if constexpr (std::is_same<QT, TagBf16>::value) {
            float top = 0.f;
#pragma unroll 1
            for (int c0 = 0; c0 < D / 8; c0 += 8) {
              uint4 x[8];
#pragma unroll
              for (int c = 0; c < 8; ++c) x[c] = src[c0 + c];
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                const uint32_t m01 = absmax_bf16x2(absmax_bf16x2(0u, x[c].x), x[c].y), m = absmax_bf16x2(absmax_bf16x2(m01, x[c].z), x[c].w);
                top = fmaxf(top, fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u)));
              }
            }
            to_f16 = row_shift(top);
          }
          const float factor = scale * p.k_scale[u.head];
          const uint32_t sign = factor < 0.f ? 0x80008000u : 0u;
          scale = fabsf(factor) / to_f16.a / to_f16.b;
          if (kWide || w == 0) {
#pragma unroll 1
            for (int c0 = 0; c0 < D / 8; c0 += 4) {
              uint4 x[4];
#pragma unroll
              for (int c = 0; c < 4; ++c) x[c] = src[c0 + c];
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                uint4 y = x[c];
                if constexpr (std::is_same<QT, TagBf16>::value)
                  y = make_uint4(bf16x2_shifted(y.x, to_f16), bf16x2_shifted(y.y, to_f16), bf16x2_shifted(y.z, to_f16), bf16x2_shifted(y.w, to_f16));
                y.x ^= sign, y.y ^= sign, y.z ^= sign, y.w ^= sign;
                *reinterpret_cast<uint4*>(dst + ((c0 + c) >> 3) * kSub + swizzled_offset(r, ((c0 + c) & 7) * 16, 128)) = y;
              }
            }
          }
        } else if (kWide || w == 0) {
          uint4 x[D / 8];
#pragma unroll
          for (int c = 0; c < D / 8; ++c) x[c] = src[c];
#pragma unroll
          for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4*>(dst + (c >> 3) * kSub + swizzled_offset(r, (c & 7) * 16, 128)) = x[c];
        }
      }
      if (kWide || w == 0) {
        fence_async_smem();
        mbar_arrive_warp(&s.q_full);
      }
      ++units;
      float m = -INFINITY, l = 0.f;
      for (int step = 0; step < n_steps; ++step) {
        const int buf = step & 1;
        mbar_wait_warp(&s.s_full[w][buf], phases >> buf & 1u, &s.abort_flag, p.status, 18);
        phases ^= 1u << buf;
        tc_fence_after();
        if (active) {
          const int keys = step_keys<kWide>(piece, w, step);
          uint64_t* before = &s.o_done[w][buf ^ 1];
          const uint32_t parity_before = (phases >> (buf ^ 1) & 1u) ^ 1u;
          if (keys == kStep)
            softmax_step<D, Mma, kE4M3, true>(ts + buf * kStep, to, keys, scale, m, l, s, before, parity_before, step == 0, p.status);
          else
            softmax_step<D, Mma, kE4M3, false>(ts + buf * kStep, to, keys, scale, m, l, s, before, parity_before, step == 0, p.status);
        }
        tc_fence_before();
        mbar_arrive_warp(&s.p_ready[w][buf]);
      }
      // ---- the piece goes to its slot
      const int64_t slot = (int64_t)u.index + blockIdx.x;
      const int64_t at = slot * p.prefix_rows + (kWide ? row : r);
      float* out = p.prefix_acc + at * D;
      const int other = kWide ? 0 : (piece - (w ^ 1) * kStep + kPrefixTile - 1) / kPrefixTile;
      other_phases ^= (uint32_t)((other + 1) / 2 & 1) | (uint32_t)(other / 2 & 1) << 1;
      if (kWide || two) {
        const int last = (n_steps - 1) & 1;
        if (n_steps > 0) mbar_wait_warp(&s.o_done[w][last], (phases >> last & 1u) ^ 1u, &s.abort_flag, p.status, 20);
        tc_fence_after();
        if (active) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(to + c, o);
            tmem_ld_wait(o);
            if (n_steps == 0)  // a piece without keys for this half
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = 0u;
            if (there)
#pragma unroll
              for (int j = 0; j < 32; j += 8) store8(out + c + j, o + j);
          }
          if (there) p.prefix_ml[at] = make_float2(m, l);
        }
        tc_fence_before();
      } else {
        // both halves hold sums of the same rows: each joins one half of the columns
        s.ml[w][r] = make_float2(m, l);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const float2 x = s.ml[w ^ 1][r];
        const bool both = w == 0 ? other > 0 : n_steps > 0;  // the second half has keys of the piece
        const int last = (n_steps - 1) & 1, other_last = (other - 1) & 1;
        if (n_steps > 0) mbar_wait_warp(&s.o_done[w][last], (phases >> last & 1u) ^ 1u, &s.abort_flag, p.status, 21);
        if (other > 0) mbar_wait_warp(&s.o_done[w ^ 1][other_last], (other_phases >> other_last & 1u) ^ 1u, &s.abort_flag, p.status, 22);
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
          if (there && w == 0) p.prefix_ml[at] = make_float2(top, l * mine + x.y * theirs);
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
  using Smem = PrefixSmem<D, kE4M3, kWide>;
  constexpr int smem = PrefixSmem<D, kE4M3, kWide>::kUsed;
  static_assert(smem >= (int)offsetof(Smem, abort_flag) + 4 && smem <= 227 * 1024, "shared memory of one CTA");
  static_assert(PrefixSmem<D, kE4M3, kWide>::kRing >= 3, "two tiles under way and one on its way");
  static std::atomic<uint64_t> allowed{0};
  if (int s = allow_smem(kernel, smem, allowed)) return s;
  FA4B_CUDA(launch_overlapped(kernel, p.prefix_workers, prefix_threads(kE4M3), smem, st, p, mk, mv));
  return FA4B_OK;
}

template <int D, bool kE4M3, typename QT>
static int launch_prefix_wide(const PagedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  if constexpr (paged_prefix_wide(D, kE4M3)) return launch_prefix_of<D, kE4M3, QT, true>(p, mk, mv, st);
  else return p.prefix_rows == 256 ? launch_prefix_of<D, kE4M3, QT, true>(p, mk, mv, st) : launch_prefix_of<D, kE4M3, QT, false>(p, mk, mv, st);
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
