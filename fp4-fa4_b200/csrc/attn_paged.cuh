// Attention over a paged cache: what the launches of one call share.
//
// A call has two kinds of work.  "Own" units: one sequence, one kv head, up to own_rows of its T x (Hq / Hkv) query rows,
// over the keys that are the sequence's own.  "Prefix" units: one group, one kv head, up to prefix_rows of the group's
// rows, over the keys that its members share, so that those are read once for all of them.  Either kind's units are
// laid end to end as one line of tiles of keys, and the line is cut into pieces of equal length, one per worker (a warp, or a
// CTA): long and short sequences load every SM alike.  What a worker has of a
// unit goes to a slot of its own (unit + worker: either grows along the line, so the sum names the pair).  The last launch
// joins the slots of a row: out = sum 2^(m_i - M) acc_i / sum 2^(m_i - M) l_i.
#pragma once
#include "attn.cuh"
#include "kv_cache.cuh"

#include <type_traits>

namespace fa4b {

constexpr int kPagedBox = 64;         // tokens of a page that one copy brings at most
constexpr int kPagedPrefixTile = 128; // keys of a tile of the prefix units
constexpr int kPagedAlign = 16;       // the shared part of a group ends on a multiple of this
constexpr int kPagedMaxRows = 4096;   // sequences of one call
constexpr int kPagedMaxT = 16;

// What the plan writes down: a worker finds its first unit in one round of loads for up to 32 sequences (two for 1024), and
// has its record in one more.
struct PagedSeq {    // one row of the batch
  int slot, len, first, cum;             // first key that is its own; length of the line before it, of one (kv head, row block)
  int g_row, g_blocks, g_unit, g_cum;  // its group's first row, row blocks, first unit, length of the line before it
  int left_alone, g_rows, pad[2];       // 1: in no group; query rows of its group, per kv head
};
struct PagedGroup {
  int shared, slot, row, rows;           // keys; whose row of the table names the pages; first row of the batch, query rows per kv head
  int cum, unit, blocks, pad;
};
// How a line is cut: at multiples of `per`.  Either every unit begins at one (`whole`: a unit's length is rounded up to pieces,
// and no piece has parts of two), or units follow one another with `extra` positions before the tiles of each.
struct PagedCut {
  uint32_t per, extra, whole;
  __device__ __forceinline__ uint32_t length(uint32_t tiles) const {  // of a unit on the line
    return tiles == 0u ? 0u : whole ? (tiles + per - 1u) / per * per : tiles + extra;
  }
};
struct PagedLine {
  uint32_t total;
  PagedCut cut;
};
struct PagedHead {
  PagedLine own, prefix;
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
  int flags;          // FA4B_PAGED_CLEAR_*
  const int32_t* seqs;
  const int32_t* offsets;
  const int32_t* shared;
  float scale_log2;
  const float* k_scale;  // this layer's [Hkv], or NULL
  const float* v_scale;
  int small;             // 1: few rows and no groups, no launch for the plan: the own units work it out
  PagedHead* head;       // the plan
  PagedSeq* seq;         // [n]
  PagedGroup* group;     // [groups]
  int* own_cum;          // [n] the line before each sequence, of one unit of each
  int* g_cum;            // [groups] the line before each group
  float* own_acc;        // [slots][own_rows][D]
  float2* own_ml;        // [slots][own_rows]: running maximum (log2 domain), sum
  float* prefix_acc;
  float2* prefix_ml;
  int own_rows, own_blocks, own_tile, own_extra, own_min, own_workers;  // rows of a unit, units per (sequence, kv head), keys of
                         // a tile, what a unit costs beside its tiles, the shortest piece, pieces
  int own_shift, own_rows_shift, own_units;             // log2 of own_tile and own_rows; units of a sequence
  int prefix_rows, prefix_shift, prefix_extra, prefix_workers;  // prefix_shift: log2 of prefix_rows
  uint32_t* status;
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }
__device__ __forceinline__ int own_tiles(const PagedParams& p, int first, int len) {
  return len > first ? ((len + p.own_tile - 1) >> p.own_shift) - (first >> p.own_shift) : 0;
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
// 2^14..2^15; a row of zeros, subnormals or infinities stays as it is).
struct RowShift {
  float a, b;  // the power of two in two steps: it may be beyond the range of one float
};
__device__ __forceinline__ RowShift row_shift(float top) {
  const int e = (int)(__float_as_uint(top) >> 23);
  const int shift = (e == 0 || e == 255) ? 0 : 127 + 14 - e;
  return {__uint_as_float((uint32_t)(127 + shift / 2) << 23), __uint_as_float((uint32_t)(127 + shift - shift / 2) << 23)};
}
__device__ __forceinline__ uint32_t bf16x2_shifted(uint32_t x, RowShift s) {  // two values of such a row
  const float2 f = unpack16(x, TagBf16{});
  return pack16(f.x * s.a * s.b, f.y * s.a * s.b, TagF16{});
}

// eight neighbours in one 32-byte store
__device__ __forceinline__ void store8(float* to, const uint32_t* x) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]),
               "r"(x[6]), "r"(x[7])
               : "memory");
}

// ---- the units --------------------------------------------------------------------------------------------------------
// A worker's walk along its line.
struct PagedUnit {
  int index;        // names the slot, together with the worker
  int head, row0, rows;   // rows row0 .. row0 + rows of the unit's sequence or group
  int first_row;    // batch row of the sequence, or the group's first
  int table_slot;   // whose row of the table names the pages
  int key_lo, key_hi;     // keys that are this unit's
  int key_all;      // own units: keys from here on are hidden from some rows
  int tile, tile_end;     // tiles (counted from key 0) that this worker takes; none, when its piece only has the unit's beginning
};

// Where the own units' part of the plan lies.
struct PagedTables {
  const PagedLine* line;
  const PagedSeq* seq;
  const int* cum;
};

template <bool kPrefix>
struct PagedWalk {
  const PagedSeq* seq;  // own units
  int left;             // positions of the line to go
  int item, which, off;
  PagedCut cut;
  int a0, a1, a2, a3, b1, b2;  // the item's record

  __device__ __forceinline__ void load(const PagedParams& p) {
    const int4* r = kPrefix ? reinterpret_cast<const int4*>(p.group + item) : reinterpret_cast<const int4*>(seq + item);
    const int4 a = r[0];
    a0 = a.x, a1 = a.y, a2 = a.z, a3 = a.w;
    if constexpr (kPrefix) {
      const int4 b = r[1];
      b1 = b.y, b2 = b.z;
    }
  }
  __device__ __forceinline__ void start(const PagedParams& p, int worker, PagedTables t) {  // whole warps
    seq = t.seq;
    const int* cum = t.cum;
    const int n = kPrefix ? p.groups : p.n, lane = threadIdx.x & 31;
    // the first round does not wait for the head of the plan: 32 places at equal distances
    int step = (n + 31) >> 5, first = lane * step < n ? cum[lane * step] : INT_MAX;
    const int4 h = *reinterpret_cast<const int4*>(t.line);
    const uint32_t total = h.x;
    cut = {(uint32_t)h.y, (uint32_t)h.z, (uint32_t)h.w};
    const uint64_t from = (uint64_t)worker * cut.per;
    left = from < total ? (int)min(cut.per, total - (uint32_t)from) : 0;
    item = which = off = 0;
    if (left == 0) return;
    const uint32_t at = (uint32_t)from, x = kPrefix ? at : at / (uint32_t)p.own_units;
    int base = 0, cum_base = 0, range = n;
    for (;;) {  // the last item that begins at or before x
      const int k = 31 - __clz(__ballot_sync(0xffffffffu, (uint32_t)first <= x));
      cum_base = __shfl_sync(0xffffffffu, first, k);
      base += k * step;
      range = min(step, range - k * step);
      if (step == 1) break;
      step = (range + 31) >> 5;
      first = lane * step < range ? cum[base + lane * step] : INT_MAX;
    }
    item = base;
    load(p);
    const uint32_t length = cut.length(tiles(p)), rest = at - (uint32_t)cum_base * (kPrefix ? 1u : (uint32_t)p.own_units);
    which = (int)(rest / length);
    off = (int)(rest - which * length);
  }
  __device__ __forceinline__ int tiles(const PagedParams& p) const {
    return kPrefix ? (a0 + kPagedPrefixTile - 1) / kPagedPrefixTile : own_tiles(p, a2, a1);
  }
  __device__ __forceinline__ bool done() const { return left <= 0; }

  // the unit at hand; then the walk stands at the next one
  __device__ __forceinline__ PagedUnit next(const PagedParams& p) {
    PagedUnit u;
    const int n_tiles = tiles(p), extra = (int)cut.extra, length = (int)cut.length(n_tiles), upto = min(length, off + left);
    u.tile = max(off - extra, 0);
    u.tile_end = max(min(upto - extra, n_tiles), u.tile);
    int units;
    if constexpr (kPrefix) {
      units = p.c.heads * b2;
      u.key_lo = 0, u.key_hi = u.key_all = a0;
      u.index = b1 + which;
      u.head = b2 == 1 ? which : which / b2;
      u.row0 = (which - u.head * b2) << p.prefix_shift;
      u.rows = min(p.prefix_rows, a3 - u.row0);
      u.first_row = a2;
      u.table_slot = a1;
    } else {
      units = p.own_units;
      u.key_lo = a2, u.key_hi = a1;
      u.key_all = max(a2, a1 - (p.T - 1));
      const int skip = a2 >> p.own_shift;
      u.tile += skip, u.tile_end += skip;
      u.index = item * units + which;
      u.head = p.own_blocks == 1 ? which : which / p.own_blocks;
      u.row0 = (which - u.head * p.own_blocks) << p.own_rows_shift;
      u.rows = min(p.own_rows, p.R - u.row0);
      u.first_row = item;
      u.table_slot = a0;
    }
    left -= upto - off;
    off = 0;
    if (left > 0 && ++which == units) {
      which = 0;
      do {  // the line goes on, so there is another item with tiles
        ++item;
        load(p);
      } while (tiles(p) == 0);
    }
    return u;
  }
};

// Caches whose prefix units always have two blocks of 128 rows.
__host__ __device__ constexpr bool paged_prefix_wide(int D, bool e4m3) { return D == 128 && !e4m3; }

// A prefix unit of up to 64 rows in a CTA whose halves share 128: rows 0-63 take the first half's keys and rows 64-127, the same
// rows again, the second half's, so that the warps at work sit in different quarters of the SM.
__device__ __forceinline__ int prefix_in_two(const PagedParams& p, int rows) { return p.prefix_rows == 128 && rows <= 64; }

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
