// What the kernels of the attention over a paged cache with a shared prefix
// have in common: the segments of keys, the rows that see them, and the
// partial results that the last kernel joins.
//
// The keys of sequence s are the prefix (shared by all) and its own ones.
// For one key head, the b * tq * G queries of all sequences (G query heads a
// key head) form one block of rows against the prefix, so that each shared
// key is read once for many rows; the tq * G queries of one sequence form a
// block against its own keys. Either is cut into splits of its keys; each
// (rows, split) leaves per row the maximum m of its scaled scores, the sum l
// of exp(s - m) and the unnormalised output, in float32, and
//   M = max m,  out = sum_p exp(m_p - M) o_p / sum_p exp(m_p - M) l_p
// joins them in a fixed order.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "sb_cache.h"
#include "sb_ptx.cuh"

namespace sb {

// How the prefix's work is cut: items (key head, tile of rows) of `tiles` key
// tiles each, one after the other, in runs of `per_cta` key tiles a block,
// whatever items a run touches. Block b leaves parts (b - first(i)) * slots ..
// of item i, one for each of its slots (rows whose keys it splits once more).
struct PaPrefix {
  FastDiv row_tiles;  // of a key head
  int tile_rows, tile_keys;
  FastDiv tiles, per_cta;
  int ctas;
  int slots;
  int parts;      // most parts an item has
  // (all key tiles together stay below 2^31)
  __host__ __device__ __forceinline__ int first(int item) const {
    return per_cta(item * tiles.d);
  }
  __host__ __device__ __forceinline__ int parts_of(int item) const {
    return slots * (static_cast<int>(per_cta((item + 1) * tiles.d - 1)) - first(item) + 1);
  }
};
// The sequences' own keys: items (sequence, key head, tile of rows), each cut
// evenly into `splits`, a block each, which leaves `slots` parts.
struct PaOwn {
  FastDiv row_tiles, splits;
  int tile_rows, tile_keys, slots, parts;
};

struct PaArgs {
  const void* k;
  const void* v;
  long page_stride, row_stride, head_stride;
  int n_pages;
  FastDiv hkv, page_rows;
  const void* q;
  long ldq;
  void* out;
  long ldo;
  float* lse;
  int b, tq, hq;
  FastDiv group;     // G = hq / hkv
  FastDiv seq_rows;  // tq * G
  float scale;
  const int* prefix_pages;
  int prefix_len;
  const int* pages;
  int max_pages;
  int capacity;      // max_pages * page_rows
  const int* lens;
  PaPrefix prefix;
  PaOwn own;
  // partial results: o [parts][b * tq * hq][hd], ml [parts][b * tq * hq];
  // parts: the prefix's, then the own splits'
  float* part_o;
  float2* part_ml;
  int box_rows;      // rows of a tiled copy: a power of two that divides a page
  bool direct;       // there is one part: results go straight to out, lse
  int* err;
};

// A block of rows against a range of one segment's keys.
struct PaPiece {
  int seq;     // -1: the prefix
  int head;    // key head
  int row0;    // first of the tile's rows among the segment's
  int rows;    // the segment's rows
  int part;    // where its (first slot's) partial results go
  int k0, k1;  // keys
};

__device__ __forceinline__ int seq_len(const PaArgs& a, int s) {
  const int n = a.lens[s];
  if (n > a.capacity) {
    report_index(a.err);
    return a.capacity;
  }
  return n;
}

// Token (sequence, query) and query head of row i of a segment.
struct PaRow {
  int s, t, h;
  long token;  // s * tq + t
};
__device__ __forceinline__ PaRow row_of(const PaArgs& a, const PaPiece& w, int i) {
  PaRow r;
  int in_seq = i;
  r.s = w.seq;
  if (w.seq < 0) {
    r.s = a.seq_rows(i);
    in_seq = i - r.s * a.seq_rows.d;
  }
  r.t = a.group(in_seq);
  r.h = w.head * a.group.d + (in_seq - r.t * a.group.d);
  r.token = static_cast<long>(r.s) * a.tq + r.t;
  return r;
}

// How many of the segment's keys row r sees (the first ones).
__device__ __forceinline__ int visible(const PaArgs& a, bool prefix, const PaRow& r) {
  const int n = seq_len(a, r.s);
  if (n < 0) return 0;
  const int own = n - a.tq + r.t + 1;
  if (!prefix) return max(own, 0);
  return max(min(a.prefix_len + own, a.prefix_len), 0);
}

// The pieces of a block that takes a run of the prefix's key tiles.
struct PaRun {
  int item, tile, left;  // the next key tile and how many are left
  __device__ __forceinline__ PaRun(const PaPrefix& p, int hkv, int cta) {
    const uint32_t at = static_cast<uint32_t>(cta) * p.per_cta.d;
    const uint32_t all = static_cast<uint32_t>(hkv) * p.row_tiles.d * p.tiles.d;
    left = at < all ? static_cast<int>(min(all - at, p.per_cta.d)) : 0;
    item = p.tiles(at);
    tile = static_cast<int>(at - item * p.tiles.d);
  }
  __device__ __forceinline__ bool next(const PaArgs& a, int cta, PaPiece& w) {
    if (left <= 0) return false;
    const PaPrefix& p = a.prefix;
    const int n = min(left, static_cast<int>(p.tiles.d) - tile);
    w.seq = -1;
    w.head = p.row_tiles(item);
    w.row0 = (item - w.head * static_cast<int>(p.row_tiles.d)) * p.tile_rows;
    w.rows = a.b * a.seq_rows.d;
    w.part = (cta - p.first(item)) * p.slots;
    w.k0 = tile * p.tile_keys;
    // (an item's tiles may be counted beyond its end, to a multiple of a run)
    w.k1 = static_cast<int>(min(static_cast<long>(tile + n) * p.tile_keys, static_cast<long>(a.prefix_len)));
    left -= n;
    tile = 0;
    ++item;
    return true;
  }
};

// The piece of a block that takes a split of a sequence's own keys; row tiles
// fastest, so that blocks that run together share keys.
__device__ __forceinline__ PaPiece own_piece(const PaArgs& a, int i) {
  PaPiece w;
  const PaOwn& o = a.own;
  const int rest = o.row_tiles(i), tile = i - rest * static_cast<int>(o.row_tiles.d);
  const int split_of = a.hkv(rest);
  w.head = rest - split_of * static_cast<int>(a.hkv.d);
  w.seq = o.splits(split_of);
  const int splits = o.splits.d, split = split_of - w.seq * splits;
  w.row0 = tile * o.tile_rows;
  w.rows = a.seq_rows.d;
  w.part = a.prefix.parts + split * o.slots;
  // keys that the tile's last row sees
  const int n = max(seq_len(a, w.seq), 0);
  const int last = a.group(min(w.row0 + o.tile_rows, w.rows) - 1);  // its query
  const int len = min(n, max(n - a.tq + last + 1, 0));
  const int tiles = (len + o.tile_keys - 1) / o.tile_keys;
  w.k0 = static_cast<int>(splits == 1 ? 0 : static_cast<long>(tiles) * split / splits) * o.tile_keys;
  w.k1 = splits == 1 ? len : min(static_cast<int>(static_cast<long>(tiles) * (split + 1) / splits) * o.tile_keys, len);
  return w;
}

// Page of the segment that holds its key j.
__device__ __forceinline__ int page_of(const PaArgs& a, const int* table, int j) {
  int page = table[a.page_rows(j)];
  if (page < 0 || page >= a.n_pages) {
    report_index(a.err);
    page = 0;
  }
  return page;
}
// Element offset of key j of the segment (head 0).
__device__ __forceinline__ long key_offset(const PaArgs& a, const int* table, int j) {
  const int row = j - static_cast<int>(a.page_rows(j) * a.page_rows.d);
  return page_of(a, table, j) * a.page_stride + static_cast<long>(row) * a.row_stride;
}
__device__ __forceinline__ const int* table_of(const PaArgs& a, const PaPiece& w) {
  return w.seq < 0 ? a.prefix_pages : a.pages + static_cast<long>(w.seq) * a.max_pages;
}

// Whether a reference of exponents in log2 units lies so far out that s sl - ref,
// fused, may differ by whole numbers from what the reference's own rounding of
// the product says (beyond 2^24; by hundreds from 2^32 on, which are 0 or
// infinite weights). Scores are then scaled and rounded before the difference.
__device__ __forceinline__ bool far_out(float ref) { return ref != -INFINITY && fabsf(ref) > 4194304.f; }

bool cache_map(void* map, const void* base, const PaArgs& a, int hd);

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
}
// ... of data that is read once
__device__ __forceinline__ uint64_t read_once_policy() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool read, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src),
               "r"(read ? 16 : 0), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace sb
