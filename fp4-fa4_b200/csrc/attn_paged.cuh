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

}  // namespace fa4b
