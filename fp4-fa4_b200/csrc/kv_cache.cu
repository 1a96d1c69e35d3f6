// Pages of a key / value cache: claim, write, fork, copy, compact, free.  Everything here moves bytes; what decides the
// time is how many launches a call needs while it is small and how close the copies come to the memory's rate when it
// is large: 250 pages of 32 layers (1.05 GB read and written) take 164 us, 6.4 TB/s; a single page 2.3 us in a graph.  Claiming is deterministic (the lowest free pages, in the order of the request), so two runs of a program
// hold the same pages.
#include "kv_cache.cuh"

namespace fa4b {

// `work` behind the status words: header of a fork or compaction, a bit per slot whose last extend was refused, then the lists
// of a compaction: used pages of each block of kBlockPages, holes, movers by the used pages before them, and those per page (at least
// 3 num_pages words; claims, forks and copies keep their free pages and flags there)
constexpr int kWorkStatus = kKvStatus, kWorkHead = kKvHead, kWorkRefused = 16, kWorkLists = kWorkRefused + FA4B_KV_MAX_SEQS / 32;
constexpr int kBlockPages = 4096;  // of a compaction: 1024 threads x 4
constexpr int kPieceBytes = 32768;  // what one CTA of the copy kernels moves: 256 threads x 8 x 16 bytes, all loads in flight at once
constexpr int kWarpBytes = 4096;    // the same per warp
constexpr int kCheckInline = 1024;  // copy lists up to this length are checked for collisions by the copying CTAs themselves

enum KvFinding { kOk = 0, kNoPages = 1, kBadSlot = 2, kSlotTwice = 3, kChildInUse = 4, kRowTooShort = 5, kBadPage = 6, kBadCount = 7, kCollision = 8, kRefused = 9, kShared = 10 };

__device__ __forceinline__ void kv_report(const KvView& c, int what, int index, int detail) {
  if (atomicCAS(c.work + kWorkStatus, 0, what) == 0) {
    c.work[kWorkStatus + 1] = index;
    c.work[kWorkStatus + 2] = detail;
  }
}

// A slot whose last extend was refused: the tokens that were to follow have no place, so that a write, which goes by the length, would
// land on the tokens before them.
__device__ __forceinline__ uint32_t* refused_word(const KvView& c, int slot) { return reinterpret_cast<uint32_t*>(c.work) + kWorkRefused + (slot >> 5); }
__device__ __forceinline__ bool is_refused(const KvView& c, int slot) { return *refused_word(c, slot) >> (slot & 31) & 1u; }
__device__ __forceinline__ void mark_refused(const KvView& c, int slot) { atomicOr(refused_word(c, slot), 1u << (slot & 31)); }
__device__ __forceinline__ void clear_refused(const KvView& c, int slot) {
  if (is_refused(c, slot)) atomicAnd(refused_word(c, slot), ~(1u << (slot & 31)));
}

__device__ __forceinline__ int pages_of(const KvView& c, int len) { return (int)(((int64_t)len + c.page_tokens - 1) >> c.page_shift); }

// exclusive prefix sum over a block of 1024 threads; `total` gets the sum
__device__ __forceinline__ int block_scan1024(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  const int before = x - v + (warp ? warp_sums[warp - 1] : 0);
  total = warp_sums[31];
  __syncthreads();
  return before;
}

// sixteen counts from page `p` on as a mask of the free pages
__device__ __forceinline__ uint32_t free_mask16(const KvView& c, int64_t p) {
  int r[16];
  if (p + 16 <= c.pages) {
    const int4* q = reinterpret_cast<const int4*>(c.refs + p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int4 x = __ldcg(q + i);
      r[4 * i] = x.x, r[4 * i + 1] = x.y, r[4 * i + 2] = x.z, r[4 * i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = p + i < c.pages ? __ldcg(c.refs + p + i) : 1;
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m |= (uint32_t)(r[i] <= 0) << i;
  return m;
}

// the same for the four pages in use from `p` on
__device__ __forceinline__ uint32_t used_mask4(const KvView& c, int64_t p) {
  int4 r = make_int4(0, 0, 0, 0);
  if (p + 4 <= c.pages) {
    r = __ldcg(reinterpret_cast<const int4*>(c.refs + p));
  } else {
    if (p < c.pages) r.x = __ldcg(c.refs + p);
    if (p + 1 < c.pages) r.y = __ldcg(c.refs + p + 1);
    if (p + 2 < c.pages) r.z = __ldcg(c.refs + p + 2);
  }
  return (uint32_t)(r.x > 0) | (uint32_t)(r.y > 0) << 1 | (uint32_t)(r.z > 0) << 2 | (uint32_t)(r.w > 0) << 3;
}

// The first `want` free pages in ascending order into out[]; a block of 1024 threads looks at 16384 pages per step and
// stops as soon as it has enough.  Returns how many there are (at least `want`, when it stopped early).
__device__ int find_free(const KvView& c, int want, int32_t* out, int* warp_sums) {
  int have = 0;
  for (int64_t base = 0; base < c.pages && have < want; base += 16384) {
    const int64_t p = base + threadIdx.x * 16;
    uint32_t m = p < c.pages ? free_mask16(c, p) : 0u;
    int total;
    int rank = have + block_scan1024(__popc(m), warp_sums, total);
    while (m != 0u && rank < want) {
      out[rank++] = (int32_t)(p + __ffs(m) - 1);
      m &= m - 1;
    }
    have += total;
  }
  __syncthreads();
  return have;
}

// ---- free -------------------------------------------------------------------------------------------------------------
// One CTA per slot.  The exchange of the length decides who frees a slot that the list names twice.
__global__ void __launch_bounds__(128) kv_free_kernel(const KvView c, const int32_t* seqs) {
  pdl_trigger();
  pdl_wait();
  __shared__ int held;
  const int slot = seqs[blockIdx.x];
  if (slot < 0 || slot >= c.max_seqs) {
    if (threadIdx.x == 0) kv_report(c, kBadSlot, blockIdx.x, slot);
    return;
  }
  if (threadIdx.x == 0) {
    held = min(pages_of(c, max(atomicExch(c.lens + slot, 0), 0)), c.width);
    clear_refused(c, slot);
  }
  __syncthreads();
  int32_t* row = c.table + slot * c.table_stride;
  for (int j = threadIdx.x; j < held; j += 128) {
    const int p = row[j];
    if (p >= 0 && p < c.pages) atomicSub(c.refs + p, 1);
    row[j] = -1;
  }
}

// ---- extend -----------------------------------------------------------------------------------------------------------
// Checks a list of distinct slots against a bitmap in shared memory; true where slot i is new and in range.
__device__ __forceinline__ int check_slot(const KvView& c, int slot, uint32_t* seen) {
  if (slot < 0 || slot >= c.max_seqs) return kBadSlot;
  const uint32_t bit = 1u << (slot & 31);
  return (atomicOr(seen + (slot >> 5), bit) & bit) ? kSlotTwice : kOk;
}

// One CTA: what is claimed in one call is a few thousand pages at most, and the order of the claims is a prefix sum over
// requests and one over free pages.  Latency bounds it (a few rounds of loads and two sums: 2 to 6 us).
__global__ void __launch_bounds__(1024) kv_extend_kernel(const KvView c, const int32_t* seqs, const int32_t* n_new,
                                                         int n, int32_t* fresh) {
  extern __shared__ int dyn[];
  __shared__ int warp_sums[32];
  int* first = dyn;                                          // [n + 1]: claims before request i
  uint32_t* seen = reinterpret_cast<uint32_t*>(dyn + n + 1);  // [max_seqs / 32]
  pdl_trigger();
  for (int i = threadIdx.x; i < (c.max_seqs + 31) / 32; i += 1024) seen[i] = 0u;
  __syncthreads();
  pdl_wait();
  bool bad = false;
  int want = 0;
  for (int base = 0; base < n; base += 1024) {
    const int i = base + threadIdx.x;
    int need = 0;
    if (i < n) {
      const int slot = seqs[i], add = n_new[i];
      int e = check_slot(c, slot, seen);
      if (e == kOk) {
        const int len = c.lens[slot];
        if (add < 0) e = kBadCount;
        else if ((int64_t)len + add > (int64_t)c.width << c.page_shift || len < 0) e = kRowTooShort;
        else need = pages_of(c, len + add) - pages_of(c, len);
      }
      if (e != kOk) {
        kv_report(c, e, i, slot);
        bad = true;
      }
    }
    int total;
    const int before = block_scan1024(need, warp_sums, total);
    if (i < n) first[i] = want + before;
    want += total;  // at most 4096 x 2^18
  }
  if (threadIdx.x == 0) first[n] = want;
  bad = __syncthreads_or(bad);
  const int have = want && !bad ? find_free(c, want, fresh, warp_sums) : 0;
  if (bad || have < want) {
    if (threadIdx.x == 0 && !bad) kv_report(c, kNoPages, want, have);
    for (int i = threadIdx.x; i < n; i += 1024) {
      const int slot = seqs[i];
      if (slot >= 0 && slot < c.max_seqs) mark_refused(c, slot);
    }
    return;
  }
  for (int r = threadIdx.x; r < want; r += 1024) {
    int lo = 0, hi = n - 1;  // the last request whose claims begin at or before r
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= r) lo = mid; else hi = mid - 1;
    }
    const int slot = seqs[lo], p = fresh[r];
    c.table[slot * c.table_stride + pages_of(c, c.lens[slot]) + (r - first[lo])] = p;
    c.refs[p] = 1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += 1024) {
    const int slot = seqs[i];
    c.lens[slot] += n_new[i];
    clear_refused(c, slot);
  }
}

// ---- write ------------------------------------------------------------------------------------------------------------
struct WriteParams {
  const uint8_t* src[2];
  int64_t sb[2], sh[2], st[2];  // byte strides: batch, head, token
  const float* scale[2];        // this layer's, or NULL
  uint8_t* dst[2];              // this layer's pool
  const int32_t* seqs;
  const int32_t* n_new;
  int T, D, tile_tokens;
};

// The head's scale with its reciprocal, for the quotients of div2_exact: correctly rounded ones for a scale of ordinary size
// whose significand is not all ones (r = 0: divide).
struct QuantScale {
  float s, r;
  __device__ __forceinline__ explicit QuantScale(float scale) : s(scale) {
    const float a = fabsf(scale);
    r = a >= 5.4e-20f && a <= 1.8e19f && !significand_all_ones(scale) ? __frcp_rn(scale) : 0.f;
  }
};
template <typename Src>
__device__ __forceinline__ uint2 quantise8(uint4 x, QuantScale scale) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint64_t f[4], q[4];
  uint32_t top = 0u;  // largest magnitudes of the even and of the odd values
  const uint64_t r2 = pack2(scale.r, scale.r), neg2 = pack2(-scale.s, -scale.s);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<Src, __half>::value) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[i] = pack2(p.x, p.y);
    } else {
      f[i] = bf16x2_to_f32x2(w[i]);
      top = absmax_bf16x2(top, w[i]);
    }
    q[i] = div2_exact(f[i], r2, neg2);
  }
  float a[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2(q[i], a[2 * i], a[2 * i + 1]);
  // an odd scale, or a quotient that may overflow on the way (f16: infinity alone, whose quotient is one as well)
  const float most = std::is_same<Src, __half>::value ? 0.f : fmaxf(__uint_as_float(top << 16), __uint_as_float(top & 0xffff0000u));
  bool divide = scale.r == 0.f || !(most * fabsf(scale.r) < 1.0e30f);
  if constexpr (std::is_same<Src, __half>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) divide |= (w[i] & 0x7fffu) == 0x7c00u || (w[i] & 0x7fff0000u) == 0x7c000000u;
  }
  if (divide) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unpack2(f[i], a[2 * i], a[2 * i + 1]);
      a[2 * i] = __fdiv_rn(a[2 * i], scale.s), a[2 * i + 1] = __fdiv_rn(a[2 * i + 1], scale.s);
    }
  }
  return make_uint2(cvt_e4m3x4(a[0], a[1], a[2], a[3]), cvt_e4m3x4(a[4], a[5], a[6], a[7]));
}

// grid (row of the batch x kv head, tile of tokens); a thread takes 16 bytes of K and of V of one token at a time, so a
// warp reads 512 contiguous bytes and writes whole rows.  Bound by memory: 2 x 2 bytes read, 2 x (1 or 2) written a value.  32 rows
// of up to 2011 tokens: 46 us into bf16 (277 MB, 6.0 TB/s), 42.4 us into E4M3 (208 MB, 4.9 TB/s; it was 61 with divisions, 48 with quotients by a
// reciprocal and one correction, 41 with three CTAs per SM instead of two, before the counts of the pages were read).  80 registers a
// thread are what three CTAs leave; E4M3 has 20 bytes beyond them.
template <bool kE4M3, typename Src>
__global__ void __launch_bounds__(256, 3) kv_write_kernel(const KvView c, const WriteParams w) {
  pdl_trigger();
  pdl_wait();
  const int i = blockIdx.x / c.heads, h = blockIdx.x - i * c.heads;
  const int slot = w.seqs[i], n_new = w.n_new ? w.n_new[i] : w.T;
  const int tile0 = blockIdx.y * w.tile_tokens, t_end = min(min(n_new, w.T), tile0 + w.tile_tokens);
  if (slot < 0 || slot >= c.max_seqs) {
    if (threadIdx.x == 0 && h == 0 && blockIdx.y == 0) kv_report(c, kBadSlot, i, slot);
    return;
  }
  if (tile0 >= t_end) return;
  const int64_t start = (int64_t)c.lens[slot] - n_new;
  if (is_refused(c, slot)) {
    if (threadIdx.x == 0 && h == 0 && blockIdx.y == 0) kv_report(c, kRefused, i, slot);
    return;
  }
  const int chunks = w.D / 8, chunk = threadIdx.x & (chunks - 1), step = 256 / chunks;
  const int32_t* row = c.table + slot * c.table_stride;
  const QuantScale sk(kE4M3 ? w.scale[0][h] : 1.f), sv(kE4M3 ? w.scale[1][h] : 1.f);
  constexpr int kOut = kE4M3 ? 8 : 16;
  const uint8_t* k_src = w.src[0] + i * w.sb[0] + h * w.sh[0] + chunk * 16;
  const uint8_t* v_src = w.src[1] + i * w.sb[1] + h * w.sh[1] + chunk * 16;
  uint8_t* k_dst = w.dst[0] + (int64_t)h * c.page_tokens * c.row_bytes + chunk * kOut;
  uint8_t* v_dst = w.dst[1] + (int64_t)h * c.page_tokens * c.row_bytes + chunk * kOut;
  // four tokens per thread at a time: their pages, then all their loads, then the stores
#pragma unroll 1
  for (int t0 = tile0 + (int)(threadIdx.x / chunks); t0 < t_end; t0 += 4 * step) {
    int page[4], at[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t pos = start + t0 + j * step;
      const bool there = t0 + j * step < t_end && pos >= 0 && (pos >> c.page_shift) < c.width;
      page[j] = there ? row[(int)(pos >> c.page_shift)] : -1;
      at[j] = ((int)pos & (c.page_tokens - 1)) * c.row_bytes;
    }
    uint4 xk[4], xv[4];
    int held[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if ((uint32_t)page[j] < (uint32_t)c.pages) held[j] = c.refs[page[j]];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if ((uint32_t)page[j] < (uint32_t)c.pages) {
        xk[j] = __ldcs(reinterpret_cast<const uint4*>(k_src + (t0 + j * step) * w.st[0]));
        xv[j] = __ldcs(reinterpret_cast<const uint4*>(v_src + (t0 + j * step) * w.st[1]));
      }
    if (max(max(held[0], held[1]), max(held[2], held[3])) > 1) {  // other slots' tokens as well
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (held[j] > 1) {
          if (h == 0 && chunk == 0) kv_report(c, kShared, i, page[j]);
          page[j] = -1;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if ((uint32_t)page[j] < (uint32_t)c.pages) {
        uint8_t* dk = k_dst + page[j] * c.k_page + at[j];
        uint8_t* dv = v_dst + page[j] * c.v_page + at[j];
        if constexpr (kE4M3) {
          *reinterpret_cast<uint2*>(dk) = quantise8<Src>(xk[j], sk);
          *reinterpret_cast<uint2*>(dv) = quantise8<Src>(xv[j], sv);
        } else {
          *reinterpret_cast<uint4*>(dk) = xk[j];
          *reinterpret_cast<uint4*>(dv) = xv[j];
        }
      }
  }
}

// ---- fork -------------------------------------------------------------------------------------------------------------
// First launch, one CTA: checks the lists, claims the tail pages and puts them into the children's rows; head[0]: 1 when the second
// launch may go on.
__global__ void __launch_bounds__(1024) kv_fork_plan_kernel(const KvView c, const int32_t* parents, const int32_t* children,
                                                            int n, int32_t* list) {
  extern __shared__ uint32_t seen[];  // [max_seqs / 32]
  __shared__ int warp_sums[32];
  constexpr int kEach = FA4B_KV_MAX_LIST / 1024;
  int rank[kEach];  // of the tail pages of this thread's children among all; -1: none
  pdl_trigger();
  for (int i = threadIdx.x; i < (c.max_seqs + 31) / 32; i += 1024) seen[i] = 0u;
  __syncthreads();
  pdl_wait();
  if (threadIdx.x == 0) c.work[kWorkHead] = 0;
  bool bad = false;
  int want = 0;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = k * 1024 + threadIdx.x;
    rank[k] = -1;
    if (k * 1024 >= n) continue;
    int need = 0;
    if (i < n) {
      const int parent = parents[i], child = children[i];
      int e = check_slot(c, child, seen), named = child;
      if (e == kOk && (parent < 0 || parent >= c.max_seqs)) e = kBadSlot, named = parent;
      if (e == kOk && c.lens[child] != 0) e = kChildInUse;
      if (e == kOk) {
        const int len = c.lens[parent];
        if (len < 0 || len > (int64_t)c.width << c.page_shift) e = kRowTooShort, named = parent;
        else need = (len & (c.page_tokens - 1)) != 0;
      }
      if (e != kOk) {
        kv_report(c, e, i, named);
        bad = true;
      }
    }
    int total;
    const int before = block_scan1024(need, warp_sums, total);
    if (need) rank[k] = want + before;
    want += total;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n && !bad; i += 1024) {  // an empty slot that is forked from and into at once
    const int parent = parents[i];
    if (seen[parent >> 5] >> (parent & 31) & 1u) {
      kv_report(c, kSlotTwice, i, parent);
      bad = true;
    }
  }
  if (__syncthreads_or(bad)) return;
  const int have = want ? find_free(c, want, list, warp_sums) : 0;
  if (have < want) {
    if (threadIdx.x == 0) kv_report(c, kNoPages, want, have);
    return;
  }
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = k * 1024 + threadIdx.x;
    if (i >= n) break;
    const int child = children[i], len = c.lens[parents[i]];
    if (rank[k] >= 0) {
      const int p = list[rank[k]];
      c.table[child * c.table_stride + (len >> c.page_shift)] = p;
      c.refs[p] = 1;
    }
    c.lens[child] = len;
    clear_refused(c, child);
  }
  if (threadIdx.x == 0) c.work[kWorkHead] = 1;
}

// Second launch.  CTAs 0..n-1: the child's row of the table and the counts of the pages it shares.  The others: one warp
// per 4 KB of a tail page's rows of one kv head, K or V, one layer.  Bound by memory where it is large: 256 forks of 4 layers with
// frees before them (70 MB) take 17.6 us in a graph, of which the copies take about 11; four forks take 7.9 us, three launches' latency.
__global__ void __launch_bounds__(256) kv_fork_move_kernel(const KvView c, const int32_t* parents, const int32_t* children,
                                                           int n, int pieces, int64_t units) {
  pdl_trigger();
  pdl_wait();
  if (c.work[kWorkHead] == 0) return;
  if ((int)blockIdx.x < n) {
    const int i = blockIdx.x, len = c.lens[parents[i]], full = len >> c.page_shift;
    const int32_t* from = c.table + parents[i] * c.table_stride;
    int32_t* to = c.table + children[i] * c.table_stride;
    for (int j = threadIdx.x; j < full; j += 256) {
      const int p = from[j];
      to[j] = p;
      if (p >= 0 && p < c.pages) atomicAdd(c.refs + p, 1);
    }
    return;
  }
  int64_t u = (int64_t)(blockIdx.x - n) * 8 + (threadIdx.x >> 5);
  if (u >= units) return;
  const int piece = (int)(u % pieces);
  u /= pieces;
  const int h = (int)(u % c.heads);
  u /= c.heads;
  const bool is_v = u & 1;
  u >>= 1;
  const int layer = (int)(u % c.layers), i = (int)(u / c.layers);
  const int len = c.lens[parents[i]];
  const int bytes = (len & (c.page_tokens - 1)) * c.row_bytes - piece * kWarpBytes;  // of this head's rows, from this piece on
  if (bytes <= 0) return;
  const int src = c.table[parents[i] * c.table_stride + (len >> c.page_shift)], dst = c.table[children[i] * c.table_stride + (len >> c.page_shift)];
  if (src < 0 || src >= c.pages) return;
  uint8_t* base = (is_v ? c.v : c.k) + layer * (is_v ? c.v_layer : c.k_layer) + (int64_t)h * c.page_tokens * c.row_bytes + piece * kWarpBytes;
  const int64_t page = is_v ? c.v_page : c.k_page;
  const uint4* from = reinterpret_cast<const uint4*>(base + src * page);
  uint4* to = reinterpret_cast<uint4*>(base + dst * page);
  uint4 r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if ((j * 32 + (int)(threadIdx.x & 31)) * 16 < bytes) r[j] = from[j * 32 + (threadIdx.x & 31)];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if ((j * 32 + (int)(threadIdx.x & 31)) * 16 < bytes) to[j * 32 + (threadIdx.x & 31)] = r[j];
}

// ---- whole pages ------------------------------------------------------------------------------------------------------
struct PieceRegs {
  uint4 r[8];
};
__device__ __forceinline__ void piece_load(PieceRegs& x, const uint8_t* from, int bytes) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if ((j * 256 + (int)threadIdx.x) * 16 < bytes) x.r[j] = __ldcs(reinterpret_cast<const uint4*>(from) + j * 256 + threadIdx.x);
}
__device__ __forceinline__ void piece_store(const PieceRegs& x, uint8_t* to, int bytes) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if ((j * 256 + (int)threadIdx.x) * 16 < bytes) __stcs(reinterpret_cast<uint4*>(to) + j * 256 + threadIdx.x, x.r[j]);
}

__device__ __forceinline__ bool collides(int i, int j, int s, int d, int sj, int dj) { return (j != i && dj == d) || sj == d || dj == s; }

// one warp per pair
__global__ void __launch_bounds__(256) kv_copy_check_kernel(const KvView c, const int32_t* src, const int32_t* dst, int n, int32_t* flags) {
  pdl_trigger();
  pdl_wait();
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= n) return;
  const int s = src[i], d = dst[i];
  bool bad = false;
  if (s >= 0 && d >= 0)
    for (int j = threadIdx.x & 31; j < n; j += 32) bad |= collides(i, j, s, d, src[j], dst[j]);
  bad = __any_sync(0xffffffffu, bad);
  if ((threadIdx.x & 31) == 0) flags[i] = bad;
}

// One CTA per 32 KB of a page of one layer, K or V: every thread has eight 16-byte loads in flight before its first store.  Bound by
// memory: 6.4 TB/s for 1.05 GB.
// Up to kCheckInline pairs each CTA checks its own pair (up to eight words per thread while the loads are on their way), above it
// a launch of its own does, which then costs less than the lists read by every CTA: 1024 pages of 1 KB in one layer take 5.7
// us this way and 8.5 us with a launch, 4096 of them in eight layers 190 and 141 us.
__global__ void __launch_bounds__(256) kv_copy_kernel(const KvView c, const int32_t* src, const int32_t* dst, int n,
                                                      int pieces, const int32_t* flags) {
  pdl_trigger();
  pdl_wait();
  int64_t u = blockIdx.x;
  const int piece = (int)(u % pieces);
  u /= pieces;
  const bool is_v = u & 1;
  u >>= 1;
  const int layer = (int)(u % c.layers), i = (int)(u / c.layers);
  const int s = src[i], d = dst[i];
  if (s < 0 || d < 0) return;
  const bool reports = threadIdx.x == 0 && layer == 0 && !is_v && piece == 0;
  if (s >= c.pages || d >= c.pages) {
    if (reports) kv_report(c, kBadPage, i, s >= c.pages ? s : d);
    return;
  }
  uint8_t* base = (is_v ? c.v : c.k) + layer * (is_v ? c.v_layer : c.k_layer) + (int64_t)piece * kPieceBytes;
  const int64_t page = is_v ? c.v_page : c.k_page;
  const int bytes = min(kPieceBytes, c.block_bytes - piece * kPieceBytes);
  PieceRegs x;
  piece_load(x, base + s * page, bytes);
  bool bad = false;
  if (flags == nullptr) {
    for (int j = threadIdx.x; j < n; j += 256) bad |= collides(i, j, s, d, src[j], dst[j]);
    bad = __syncthreads_or(bad);
  } else {
    bad = flags[i] != 0;
  }
  if (bad) {
    if (reports) kv_report(c, kCollision, i, d);
    return;
  }
  piece_store(x, base + d * page, bytes);
}

// ---- compact ----------------------------------------------------------------------------------------------------------
struct CompactLists {
  int32_t *counts, *holes, *movers, *rank;
};
__host__ __device__ inline int compact_blocks(int pages) { return (pages + kBlockPages - 1) / kBlockPages; }
__device__ __forceinline__ CompactLists compact_lists(const KvView& c) {
  CompactLists l;
  l.counts = c.work + kWorkLists;
  l.holes = l.counts + compact_blocks(c.pages);
  l.movers = l.holes + c.pages;
  l.rank = l.movers + c.pages;
  return l;
}

// used pages of each block, where there is more than one
__global__ void __launch_bounds__(1024) kv_compact_count_kernel(const KvView c) {
  pdl_trigger();
  pdl_wait();
  __shared__ int warp_sums[32];
  int total;
  block_scan1024(__popc(used_mask4(c, (int64_t)blockIdx.x * kBlockPages + threadIdx.x * 4)), warp_sums, total);
  if (threadIdx.x == 0) compact_lists(c).counts[blockIdx.x] = total;
}

// With U used pages in all and b(p) used pages below p: a free page p < U is hole p - b(p); a used page p >= U is the
// mover after the b(p) - b(U) movers before it.  Movers are kept at b(p); head = {U, b(U)} lets the last launch pair them.
__global__ void __launch_bounds__(1024) kv_compact_plan_kernel(const KvView c) {
  pdl_trigger();
  pdl_wait();
  const CompactLists l = compact_lists(c);
  __shared__ int warp_sums[32], sums[2];
  if (threadIdx.x < 2) sums[threadIdx.x] = 0;
  const int64_t p0 = (int64_t)blockIdx.x * kBlockPages + threadIdx.x * 4;
  const uint32_t m = used_mask4(c, p0);
  int n_used;
  int b = block_scan1024(__popc(m), warp_sums, n_used);
  if (gridDim.x > 1) {
    int before = 0, used = 0;
    for (int j = threadIdx.x; j < (int)gridDim.x; j += 1024) {
      const int v = l.counts[j];
      used += v;
      before += j < (int)blockIdx.x ? v : 0;
    }
    used = __reduce_add_sync(0xffffffffu, used);
    before = __reduce_add_sync(0xffffffffu, before);
    if ((threadIdx.x & 31) == 0) atomicAdd(&sums[0], used), atomicAdd(&sums[1], before);
    __syncthreads();
    n_used = sums[0];
    b += sums[1];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t p = p0 + j;
    if (p >= c.pages) break;
    if (p == n_used) c.work[kWorkHead] = n_used, c.work[kWorkHead + 1] = b;
    if (m >> j & 1u) {
      if (p >= n_used) l.movers[b] = (int32_t)p, l.rank[p] = b;
      ++b;
    } else if (p < n_used) {
      l.holes[p - b] = (int32_t)p;
    }
  }
  if (n_used >= c.pages && blockIdx.x == 0 && threadIdx.x == 0) c.work[kWorkHead] = c.work[kWorkHead + 1] = n_used;
}

// The moves (destinations lie below U, sources at or above it, so no order matters), counts and tables.  How many there are
// only the device knows: a fixed grid walks them.  16001 pages of 4 layers, a third in use (1.74 GB read and written): 300 us for
// the call, 5.8 TB/s; 200 pages: 6.0 us, two launches' latency.
__global__ void __launch_bounds__(256) kv_compact_move_kernel(const KvView c, int pieces) {
  pdl_trigger();
  pdl_wait();
  const CompactLists l = compact_lists(c);
  const int n_used = c.work[kWorkHead], b_used = c.work[kWorkHead + 1], moves = n_used - b_used;
  const int64_t units = (int64_t)moves * c.layers * 2 * pieces;
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    int64_t u = unit;
    const int piece = (int)(u % pieces);
    u /= pieces;
    const bool is_v = u & 1;
    u >>= 1;
    const int layer = (int)(u % c.layers), i = (int)(u / c.layers);
    uint8_t* base = (is_v ? c.v : c.k) + layer * (is_v ? c.v_layer : c.k_layer) + (int64_t)piece * kPieceBytes;
    const int64_t page = is_v ? c.v_page : c.k_page;
    const int bytes = min(kPieceBytes, c.block_bytes - piece * kPieceBytes);
    PieceRegs x;
    piece_load(x, base + l.movers[b_used + i] * page, bytes);
    piece_store(x, base + l.holes[i] * page, bytes);
  }
  const int64_t tid = (int64_t)blockIdx.x * 256 + threadIdx.x, threads = (int64_t)gridDim.x * 256;
  for (int64_t i = tid; i < moves; i += threads) {
    const int from = l.movers[b_used + i];
    c.refs[l.holes[i]] = c.refs[from];
    c.refs[from] = 0;
  }
  if (moves == 0) return;
  // a warp per slot's row, entries of the slot's length only
  for (int64_t s = tid >> 5; s < c.max_seqs; s += threads >> 5) {
    const int held = min(pages_of(c, max(c.lens[s], 0)), c.width);
    int32_t* row = c.table + s * c.table_stride;
    for (int j = threadIdx.x & 31; j < held; j += 32) {
      const int p = row[j];
      if (p < n_used || p >= c.pages) continue;
      const int i = l.rank[p] - b_used;  // of a page that no count covers this is what some earlier call left: not followed
      if (i >= 0 && i < moves && l.movers[b_used + i] == p) row[j] = l.holes[i];
    }
  }
}

// ---- host -------------------------------------------------------------------------------------------------------------
int kv_view(const fa4b_kv_cache* c, KvView* out) {
  FA4B_REQUIRE(c != nullptr, FA4B_BAD_ARG, "cache is NULL");
  FA4B_REQUIRE(c->dtype == FA4B_KV_BF16 || c->dtype == FA4B_KV_F16 || c->dtype == FA4B_KV_E4M3, FA4B_UNSUPPORTED, "unknown cache dtype %d", c->dtype);
  FA4B_REQUIRE(c->D == 64 || c->D == 128, FA4B_BAD_SHAPE, "head dim %d: only 64 and 128 are built", c->D);
  FA4B_REQUIRE(c->page_tokens == 16 || c->page_tokens == 32 || c->page_tokens == 64 || c->page_tokens == 128, FA4B_BAD_SHAPE,
               "pages of %d tokens: 16, 32, 64 or 128 are built", c->page_tokens);
  FA4B_REQUIRE(c->layers > 0 && c->num_pages > 0 && c->Hkv > 0 && c->max_seqs > 0 && c->table_width > 0, FA4B_BAD_SHAPE,
               "layers, num_pages, Hkv, max_seqs and table_width must be positive");
  FA4B_REQUIRE(c->max_seqs <= FA4B_KV_MAX_SEQS, FA4B_BAD_SHAPE, "max_seqs=%d is above %d", c->max_seqs, (int)FA4B_KV_MAX_SEQS);
  FA4B_REQUIRE(c->table_width <= (1 << 18) && c->Hkv <= 1024 && c->layers <= 4096 && c->num_pages <= 1 << 30, FA4B_BAD_SHAPE,
               "table_width <= 2^18, Hkv <= 1024, layers <= 4096 and num_pages <= 2^30 are built");
  const int esz = c->dtype == FA4B_KV_E4M3 ? 1 : 2;
  const int64_t block = (int64_t)c->Hkv * c->page_tokens * c->D;
  FA4B_REQUIRE(c->k && c->v && c->page_table && c->seq_lens && c->ref_counts && c->work, FA4B_BAD_ARG, "NULL buffer in the cache");
  FA4B_REQUIRE(c->dtype != FA4B_KV_E4M3 || (c->k_scale && c->v_scale), FA4B_BAD_ARG, "an E4M3 cache needs k_scale and v_scale");
  FA4B_REQUIRE(!misaligned(c->k, 16) && !misaligned(c->v, 16) && !misaligned(c->ref_counts, 16) && !misaligned(c->work, 16), FA4B_BAD_ALIGN,
               "k, v, ref_counts and work must be 16-byte aligned");
  FA4B_REQUIRE(c->table_stride >= c->table_width || c->max_seqs == 1, FA4B_BAD_SHAPE, "rows of the page table overlap (stride %lld, width %d)",
               (long long)c->table_stride, c->table_width);
  const int64_t strides[4] = {c->k_layer_stride, c->k_page_stride, c->v_layer_stride, c->v_page_stride};
  for (int64_t s : strides)
    FA4B_REQUIRE(s >= 0 && s * esz % 16 == 0, FA4B_BAD_ALIGN, "layer and page strides must be multiples of 16 bytes");
  FA4B_REQUIRE(c->num_pages == 1 || (c->k_page_stride >= block && c->v_page_stride >= block), FA4B_BAD_SHAPE, "pages overlap: the page stride is below %lld",
               (long long)block);
  FA4B_REQUIRE(c->layers == 1 || (c->k_layer_stride >= block && c->v_layer_stride >= block), FA4B_BAD_SHAPE, "layers overlap: the layer stride is below %lld",
               (long long)block);
  KvView v{};
  v.k = static_cast<uint8_t*>(c->k);
  v.v = static_cast<uint8_t*>(c->v);
  v.k_layer = c->k_layer_stride * esz, v.k_page = c->k_page_stride * esz;
  v.v_layer = c->v_layer_stride * esz, v.v_page = c->v_page_stride * esz;
  v.layers = c->layers, v.pages = c->num_pages, v.heads = c->Hkv, v.page_tokens = c->page_tokens;
  v.page_shift = __builtin_ctz((unsigned)c->page_tokens);
  v.row_bytes = c->D * esz;
  v.block_bytes = (int)(block * esz);
  v.table = c->page_table, v.table_stride = c->table_stride, v.max_seqs = c->max_seqs, v.width = c->table_width;
  v.lens = c->seq_lens, v.refs = c->ref_counts, v.work = static_cast<int32_t*>(c->work);
  *out = v;
  return FA4B_OK;
}

// Do blocks of `block` elements at l * layer + p * page, l < layers and p < pages, keep off one another?  Both strides are `block` at least.
static bool blocks_apart(int64_t layer, int64_t page, int64_t layers, int64_t pages, int64_t block) {
  if (layers == 1 || pages == 1 || layer >= (pages - 1) * page + block || page >= (layers - 1) * layer + block) return true;  // nested either way
  for (int64_t d = 1; d < layers; ++d) {  // layers d apart: the pages that come nearest
    const int64_t at = d * layer, p = std::min(at / page, pages - 1);
    if (at - p * page < block || (p + 1 < pages && (p + 1) * page - at < block)) return false;
  }
  return true;
}

// the same for calls that write pages
static int kv_pools(const fa4b_kv_cache* c, KvView* out) {
  if (int s = kv_view(c, out)) return s;
  const int64_t block = (int64_t)c->Hkv * c->page_tokens * c->D;
  FA4B_REQUIRE(blocks_apart(c->k_layer_stride, c->k_page_stride, c->layers, c->num_pages, block) &&
                   blocks_apart(c->v_layer_stride, c->v_page_stride, c->layers, c->num_pages, block),
               FA4B_BAD_SHAPE, "layers overlap: a page of one lies on a page of another");
  return FA4B_OK;
}

static int check_list(const void* a, const void* b, int32_t n) {
  FA4B_REQUIRE(n >= 0 && n <= FA4B_KV_MAX_LIST, FA4B_BAD_SHAPE, "lists of 0 to %d entries are built, got %d", (int)FA4B_KV_MAX_LIST, n);
  FA4B_REQUIRE(n == 0 || (a && b), FA4B_BAD_ARG, "NULL list");
  return FA4B_OK;
}

}  // namespace fa4b

using namespace fa4b;

extern "C" {

size_t fa4b_kv_workspace_bytes(const fa4b_kv_cache* c) {
  if (c == nullptr || c->num_pages <= 0) return 0;
  return 4 * ((size_t)kWorkLists + compact_blocks(c->num_pages) + 3 * (size_t)c->num_pages);
}

int fa4b_kv_free(const fa4b_kv_cache* c, const int32_t* seqs, int32_t n, void* stream) {
  KvView v;
  if (int s = kv_view(c, &v)) return s;
  if (int s = check_list(seqs, seqs, n)) return s;
  if (n == 0) return FA4B_OK;
  FA4B_CUDA(launch_overlapped(kv_free_kernel, n, 128, 0, static_cast<cudaStream_t>(stream), v, seqs));
  return FA4B_OK;
}

int fa4b_kv_extend(const fa4b_kv_cache* c, const int32_t* seqs, const int32_t* n_new, int32_t n, void* stream) {
  KvView v;
  if (int s = kv_view(c, &v)) return s;
  if (int s = check_list(seqs, n_new, n)) return s;
  if (n == 0) return FA4B_OK;
  const size_t smem = 4 * ((size_t)n + 1 + (v.max_seqs + 31) / 32);
  static std::atomic<uint64_t> allowed{0};
  if (smem > kSmemUnasked)
    if (int s = allow_smem(kv_extend_kernel, 4 * (FA4B_KV_MAX_LIST + 1 + FA4B_KV_MAX_SEQS / 32), allowed)) return s;
  int32_t* fresh = v.work + kWorkLists;  // the lists of a compaction are at least num_pages long
  FA4B_CUDA(launch_overlapped(kv_extend_kernel, 1, 1024, smem, static_cast<cudaStream_t>(stream), v, seqs, n_new, n, fresh));
  return FA4B_OK;
}

int fa4b_kv_write(const fa4b_kv_cache* c, const fa4b_kv_write_args* a, void* stream) {
  KvView v;
  if (int s = kv_pools(c, &v)) return s;
  FA4B_REQUIRE(a != nullptr, FA4B_BAD_ARG, "args is NULL");
  if (int s = check_list(a->seqs, a->seqs, a->n)) return s;
  FA4B_REQUIRE(a->T >= 0, FA4B_BAD_SHAPE, "T=%d is negative", a->T);
  FA4B_REQUIRE(a->layer >= 0 && a->layer < c->layers, FA4B_BAD_SHAPE, "layer %d of %d", a->layer, c->layers);
  FA4B_REQUIRE(a->src_dtype == FA4B_KV_BF16 || a->src_dtype == FA4B_KV_F16, FA4B_UNSUPPORTED, "values are written from bf16 or f16");
  FA4B_REQUIRE(c->dtype == FA4B_KV_E4M3 || a->src_dtype == c->dtype, FA4B_UNSUPPORTED, "a 16-bit cache takes values of its own type");
  if (a->n == 0 || a->T == 0) return FA4B_OK;
  FA4B_REQUIRE(a->k_new && a->v_new, FA4B_BAD_ARG, "k_new or v_new is NULL");
  FA4B_REQUIRE(!misaligned(a->k_new, 16) && !misaligned(a->v_new, 16), FA4B_BAD_ALIGN, "k_new and v_new must be 16-byte aligned");
  const fa4b_strides st[2] = {a->k_strides, a->v_strides};
  WriteParams w{};
  w.src[0] = static_cast<const uint8_t*>(a->k_new), w.src[1] = static_cast<const uint8_t*>(a->v_new);
  for (int i = 0; i < 2; ++i) {
    FA4B_REQUIRE(st[i].batch % 8 == 0 && st[i].head % 8 == 0 && st[i].seq % 8 == 0, FA4B_BAD_ALIGN, "strides must be multiples of 8 elements");
    w.sb[i] = st[i].batch * 2, w.sh[i] = st[i].head * 2, w.st[i] = st[i].seq * 2;
  }
  if (c->dtype == FA4B_KV_E4M3) w.scale[0] = c->k_scale + (int64_t)a->layer * c->Hkv, w.scale[1] = c->v_scale + (int64_t)a->layer * c->Hkv;
  w.dst[0] = v.k + a->layer * v.k_layer, w.dst[1] = v.v + a->layer * v.v_layer;
  w.seqs = a->seqs, w.n_new = a->n_new, w.T = a->T, w.D = c->D;
  // four tokens of K and V in flight per thread; twice over where there are CTAs enough without (E4M3, 8 kv heads, D 128: 32
  // rows of up to 2011 tokens 47.8 against 51.9 us with the claims, 8 rows 14.4 against 15.6, but 4 rows 13.1 against 11.0)
  w.tile_tokens = 4 * (256 / (c->D / 8));
  if ((int64_t)a->n * c->Hkv * a->T > 12ll * w.tile_tokens * std::max(sm_count(), 1)) w.tile_tokens *= 2;
  const int64_t tiles = ((int64_t)a->T + w.tile_tokens - 1) / w.tile_tokens;
  FA4B_REQUIRE(tiles <= 65535, FA4B_BAD_SHAPE, "T=%d: at most %d tokens in one call", a->T, 65535 * w.tile_tokens);
  const dim3 grid((unsigned)(a->n * c->Hkv), (unsigned)tiles);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c->dtype != FA4B_KV_E4M3) FA4B_CUDA(launch_overlapped(kv_write_kernel<false, __nv_bfloat16>, grid, 256, 0, s, v, w));
  else if (a->src_dtype == FA4B_KV_F16) FA4B_CUDA(launch_overlapped(kv_write_kernel<true, __half>, grid, 256, 0, s, v, w));
  else FA4B_CUDA(launch_overlapped(kv_write_kernel<true, __nv_bfloat16>, grid, 256, 0, s, v, w));
  return FA4B_OK;
}

int fa4b_kv_fork(const fa4b_kv_cache* c, const int32_t* parents, const int32_t* children, int32_t n, void* stream) {
  KvView v;
  if (int s = kv_pools(c, &v)) return s;
  if (int s = check_list(parents, children, n)) return s;
  if (n == 0) return FA4B_OK;
  const int pieces = (v.page_tokens * v.row_bytes + kWarpBytes - 1) / kWarpBytes;
  const int64_t units = (int64_t)n * v.layers * 2 * v.heads * pieces, ctas = n + (units + 7) / 8;
  FA4B_REQUIRE(ctas < 1ll << 31, FA4B_BAD_SHAPE, "%d forks over %d layers and %d heads are too many for one call", n, v.layers, v.heads);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t smem = 4 * (size_t)((v.max_seqs + 31) / 32);
  FA4B_CUDA(launch_overlapped(kv_fork_plan_kernel, 1, 1024, smem, st, v, parents, children, n, v.work + kWorkLists));
  FA4B_CUDA(launch_overlapped(kv_fork_move_kernel, (unsigned)ctas, 256, 0, st, v, parents, children, n, pieces, units));
  return FA4B_OK;
}

int fa4b_kv_copy_pages(const fa4b_kv_cache* c, const int32_t* src, const int32_t* dst, int32_t n, void* stream) {
  KvView v;
  if (int s = kv_pools(c, &v)) return s;
  if (int s = check_list(src, dst, n)) return s;
  if (n == 0) return FA4B_OK;
  const int pieces = (v.block_bytes + kPieceBytes - 1) / kPieceBytes;
  const int64_t ctas = (int64_t)n * v.layers * 2 * pieces;
  FA4B_REQUIRE(ctas < 1ll << 31, FA4B_BAD_SHAPE, "%d pages of %d layers are too many for one call", n, v.layers);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // more pairs than the work area has room for flags are more than the pool has pages: few of them can be free of collisions
  int32_t* flags = n > kCheckInline && n <= 3ll * v.pages ? v.work + kWorkLists : nullptr;
  if (flags) FA4B_CUDA(launch_overlapped(kv_copy_check_kernel, (n + 7) / 8, 256, 0, st, v, src, dst, n, flags));
  FA4B_CUDA(launch_overlapped(kv_copy_kernel, (unsigned)ctas, 256, 0, st, v, src, dst, n, pieces, flags));
  return FA4B_OK;
}

int fa4b_kv_compact(const fa4b_kv_cache* c, void* stream) {
  KvView v;
  if (int s = kv_pools(c, &v)) return s;
  const int pieces = (v.block_bytes + kPieceBytes - 1) / kPieceBytes;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int blocks = compact_blocks(v.pages);
  if (blocks > 1) FA4B_CUDA(launch_overlapped(kv_compact_count_kernel, blocks, 1024, 0, st, v));
  FA4B_CUDA(launch_overlapped(kv_compact_plan_kernel, blocks, 1024, 0, st, v));
  const int64_t most = std::max<int64_t>((int64_t)(v.pages / 2) * v.layers * 2 * pieces, (v.max_seqs + 7) / 8);
  const unsigned grid = (unsigned)std::min<int64_t>(std::max<int64_t>(most, 1), (int64_t)std::max(sm_count(), 1) * 6);
  FA4B_CUDA(launch_overlapped(kv_compact_move_kernel, grid, 256, 0, st, v, pieces));
  return FA4B_OK;
}

int fa4b_kv_check_status(const fa4b_kv_cache* c, void* stream) {
  KvView v;
  if (int s = kv_view(c, &v)) return s;
  int32_t host[kKvStatusWords] = {};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  FA4B_CUDA(cudaMemcpyAsync(host, v.work + kWorkStatus, sizeof(host), cudaMemcpyDeviceToHost, st));
  FA4B_CUDA(cudaStreamSynchronize(st));
  if (host[0] == kOk && host[kKvAttnStatus] == 0) return FA4B_OK;
  // what is told now is cleared: of both kinds of findings the other waits for the next check
  const int32_t* attn = host + kKvAttnStatus;
  const bool of_attn = attn[0] == 1 || host[0] == kOk;
  FA4B_CUDA(cudaMemsetAsync(v.work + (of_attn ? kKvAttnStatus : kWorkStatus), 0, 4 * (kKvAttnStatus - kKvStatus), st));
  FA4B_REQUIRE(attn[0] != 1, FA4B_TIMEOUT, "a device-side wait of the attention over the cache ran out (site %d, block %d)", attn[1], attn[2]);
  if (host[0] == kOk && attn[0] == 3) {
    set_error("the batch's keys are too many for one call (%d tiles per kv head)", attn[1]);
    return FA4B_BAD_ARG;
  }
  if (host[0] == kOk) {
    set_error("the offsets of %d groups do not rise from 0 to at most the number of rows", attn[1]);
    return FA4B_BAD_ARG;
  }
  switch (host[0]) {
    case kNoPages: set_error("%d pages were asked for, %d are free", host[1], host[2]); return FA4B_NO_PAGES;
    case kBadSlot: set_error("entry %d names slot %d of %d", host[1], host[2], v.max_seqs); break;
    case kSlotTwice: set_error("entry %d names slot %d a second time", host[1], host[2]); break;
    case kChildInUse: set_error("entry %d forks into slot %d, which is not empty", host[1], host[2]); break;
    case kRowTooShort: set_error("entry %d: a row of the page table holds %d pages, too few for slot %d", host[1], v.width, host[2]); break;
    case kBadPage: set_error("pair %d names page %d of %d", host[1], host[2], v.pages); break;
    case kBadCount: set_error("entry %d: negative number of new tokens for slot %d", host[1], host[2]); break;
    case kRefused: set_error("entry %d writes to slot %d, whose last extend was refused", host[1], host[2]); break;
    case kShared: set_error("entry %d writes to page %d, which several slots hold", host[1], host[2]); break;
    case kCollision: set_error("pair %d: page %d is also another pair's destination or source", host[1], host[2]); break;
    default: set_error("finding %d (%d, %d)", host[0], host[1], host[2]); break;
  }
  return FA4B_BAD_ARG;
}

}  // extern "C"
