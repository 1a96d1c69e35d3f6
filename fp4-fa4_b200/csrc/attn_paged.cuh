// Attention over a paged cache: what the launches of one call share.
//
// A call has two kinds of work.  "Own" units: one sequence, one kv head, up to own_rows of its T x (Hq / Hkv) query rows,
// over the keys that are the sequence's own.  "Prefix" units: one group, one kv head, up to prefix_rows of the group's
// rows, over the keys that its members share, so that those are read once for all of them.  Either kind's units are
// laid end to end as one line of key tiles which is cut into equal pieces, one per CTA: long and short sequences load every
// SM alike, and what a CTA keeps of a unit goes to a slot of its own (unit + CTA: either grows along the line, so the sum
// names the pair).  The last launch joins the slots of a row: out = sum 2^(m_i - M) acc_i / sum 2^(m_i - M) l_i.
#pragma once
#include "attn.cuh"
#include "kv_cache.cuh"

#include <type_traits>

namespace fa4b {

constexpr int kPagedTile = 64;        // keys of a tile of the own units
constexpr int kPagedAlign = 16;       // the shared part of a group ends on a multiple of this
constexpr int kPagedMaxRows = 4096;   // sequences of one call
constexpr int kPagedMaxT = 16;

struct PagedPlan {  // device arrays in the workspace
  int* slot;        // [n] -1: none
  int* len;         // [n] keys (0: nothing to do)
  int* group;       // [n] -1: the row belongs to no group and is left alone
  int* own_cum;     // [n + 1] tiles of one (kv head, row block) before sequence i
  int* g_first;     // [groups] a member whose row of the table names the shared pages
  int* g_shared;    // [groups] shared keys that every row of the group sees
  int* g_cum;       // [groups + 1] tiles before group g, all heads and row blocks
  int* g_unit;      // [groups + 1] units before group g
};

struct PagedParams {
  KvView c;
  int layer;
  const uint8_t* q;   // 16-bit elements; strides in elements
  int64_t q_sb, q_sh, q_st;
  uint8_t* o;
  int64_t o_sb, o_sh, o_st;
  float* lse;         // [n, Hq, T]
  int n, T, Hq, G, R; // G = Hq / Hkv, R = T G rows of a sequence and kv head
  int groups;         // 0: no groups, nothing shared
  const int32_t* seqs;
  const int32_t* offsets;
  const int32_t* shared;
  float scale_log2;
  const float* k_scale;  // this layer's [Hkv], or NULL
  const float* v_scale;
  PagedPlan plan;
  float* own_acc;        // [slots][own_rows][D]
  float2* own_ml;        // [slots][own_rows]: running maximum (log2 domain), sum
  float* prefix_acc;
  float2* prefix_ml;
  int own_rows, own_blocks, own_ctas;  // rows of a unit, units per (sequence, kv head), CTAs
  int prefix_rows, prefix_tile, prefix_ctas;
  uint32_t* status;
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }
__device__ __forceinline__ int64_t piece_tiles(int64_t total, int ctas) { return total <= 0 ? 1 : (total + ctas - 1) / ctas; }

// the last i in [0, n) with cum[i] <= x (cum ascending, cum[0] = 0)
__device__ __forceinline__ int last_at_or_before(const int* cum, int n, int64_t x, int64_t factor) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int64_t)cum[mid] * factor <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int own_first_key(const PagedParams& p, int i) {
  const int g = p.plan.group[i];
  return p.groups > 0 && g >= 0 ? p.plan.g_shared[g] : 0;
}
__device__ __forceinline__ int own_tiles(int first, int len) {
  return len > first ? (len + kPagedTile - 1) / kPagedTile - first / kPagedTile : 0;
}

// ---- numbers ----------------------------------------------------------------------------------------------------------
struct TagBf16 {};
struct TagF16 {};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, TagBf16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, TagF16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, TagBf16) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, TagF16) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 unpack16(uint32_t x, TagBf16) { return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)); }
__device__ __forceinline__ float2 unpack16(uint32_t x, TagF16) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }
// two E4M3 codes -> f16 pair (exact)
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t r;
  asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.rn.f16x2.e4m3x2 %0, lo; }" : "=r"(r) : "r"(two));
  return r;
}
__device__ __forceinline__ float paged_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, int u, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
               "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(u)
               : "memory");
}


// A query row against E4M3 keys in f16: bf16 values are brought into f16's range by a power of two (the largest becomes
// 2^14..2^15; a row of zeros, subnormals or infinities stays as it is), and the sign of the factor moves into the row.
// Returns the factor, no longer negative, that undoes both.
struct RowShift {
  float a, b;  // the power of two in two steps: it may be beyond the range of one float
};
__device__ __forceinline__ RowShift row_shift(float top) {
  const int e = (int)(__float_as_uint(top) >> 23);
  const int shift = (e == 0 || e == 255) ? 0 : 127 + 14 - e;
  return {__uint_as_float((uint32_t)(127 + shift / 2) << 23), __uint_as_float((uint32_t)(127 + shift - shift / 2) << 23)};
}
template <typename QT, int kVecs>
__device__ __forceinline__ float e4m3_query_row(uint4 (&x)[kVecs], float scale) {
  const uint32_t sign = scale < 0.f ? 0x80008000u : 0u;
  scale = fabsf(scale);
  uint32_t(*w)[4] = reinterpret_cast<uint32_t(*)[4]>(x);
  if constexpr (std::is_same<QT, TagBf16>::value) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack16(w[i][j], TagBf16{});
        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
    const RowShift s = row_shift(top);
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack16(w[i][j], TagBf16{});
        w[i][j] = pack16(f.x * s.a * s.b, f.y * s.a * s.b, TagF16{});
      }
    scale = scale / s.a / s.b;
  }
#pragma unroll
  for (int i = 0; i < kVecs; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) w[i][j] ^= sign;
  return scale;
}

// eight neighbours in one 32-byte store
__device__ __forceinline__ void store8(float* to, const uint32_t* x) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]),
               "r"(x[6]), "r"(x[7])
               : "memory");
}

// ---- the units --------------------------------------------------------------------------------------------------------
// Where a CTA stands on the line of tiles.
struct PagedUnit {
  int index;        // names the slot, together with the CTA
  int head, row0, rows;   // rows row0 .. row0 + rows of the unit's sequence or group
  int first_row;    // batch row of the sequence, or the group's first
  int table_slot;   // whose row of the table names the pages
  int key_lo, key_hi;     // keys that are this unit's
  int key_all;      // own units: keys from here on are hidden from some rows
  int tile, tile_end;     // tiles (64 keys, counted from key 0) that this CTA takes
};

template <bool kPrefix>
__device__ __forceinline__ int64_t line_total(const PagedParams& p) {
  return kPrefix ? (int64_t)p.plan.g_cum[p.groups] : (int64_t)p.plan.own_cum[p.n] * p.c.heads * p.own_blocks;
}

// the unit at position `at` of the line, cut at `end`
template <bool kPrefix>
__device__ __forceinline__ PagedUnit unit_at(const PagedParams& p, int64_t at, int64_t end) {
  PagedUnit u;
  if constexpr (kPrefix) {
    const int g = last_at_or_before(p.plan.g_cum, p.groups, at, 1);
    u.key_lo = 0, u.key_hi = u.key_all = p.plan.g_shared[g];
    const int tiles = ceil_div(u.key_hi, p.prefix_tile);
    const int lo = max(p.offsets[g], 0), hi = min(p.offsets[g + 1], p.n);
    const int blocks = ceil_div((hi - lo) * p.R, p.prefix_rows);
    const int64_t off = at - p.plan.g_cum[g];
    const int which = (int)(off / tiles);
    u.tile = (int)(off % tiles);
    u.tile_end = (int)min((int64_t)tiles, u.tile + (end - at));
    u.index = p.plan.g_unit[g] + which;
    u.head = which / blocks;
    u.row0 = (which % blocks) * p.prefix_rows;
    u.rows = min(p.prefix_rows, (hi - lo) * p.R - u.row0);
    u.first_row = lo;
    u.table_slot = p.plan.slot[p.plan.g_first[g]];
  } else {
    const int per = p.c.heads * p.own_blocks;
    const int i = last_at_or_before(p.plan.own_cum, p.n, at, per);
    u.key_lo = own_first_key(p, i), u.key_hi = p.plan.len[i];
    u.key_all = max(u.key_lo, u.key_hi - (p.T - 1));
    const int tiles = own_tiles(u.key_lo, u.key_hi), skip = u.key_lo / kPagedTile;
    const int64_t off = at - (int64_t)p.plan.own_cum[i] * per;
    const int which = (int)(off / tiles);
    const int t = (int)(off % tiles);
    u.tile = skip + t;
    u.tile_end = skip + (int)min((int64_t)tiles, t + (end - at));
    u.index = i * per + which;
    u.head = which / p.own_blocks;
    u.row0 = (which % p.own_blocks) * p.own_rows;
    u.rows = min(p.own_rows, p.R - u.row0);
    u.first_row = i;
    u.table_slot = p.plan.slot[i];
  }
  return u;
}

// a row of a unit: batch row, token and query head
struct PagedRow {
  int i, t, h;
};
__device__ __forceinline__ PagedRow paged_row(const PagedParams& p, const PagedUnit& u, int row) {
  const int r = u.row0 + row, in_seq = r % p.R;
  return {u.first_row + r / p.R, in_seq / p.G, u.head * p.G + in_seq % p.G};
}

int launch_prefix(const PagedParams& p, int D, bool e4m3, bool q_f16, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st);

}  // namespace fa4b
