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

// Division of a non-negative 31-bit number by a fixed d >= 1: n / d =
// (n * mul) >> 32 >> shift with mul = floor(2^(32 + shift) / d) + 1, 2^shift
// the power of two just below d (exact for n < 2^31; Granlund and Montgomery,
// PLDI 1994).
struct FastDiv {
  uint32_t d, mul, shift;
  static FastDiv of(uint32_t d) {
    FastDiv f{d, 0, 0};
    if (d == 1) return f;
    while ((2u << f.shift) < d) ++f.shift;
    f.mul = static_cast<uint32_t>(((1ull << (32 + f.shift)) / d) + 1);
    return f;
  }
  __host__ __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
    if (d == 1) return n;
    return static_cast<uint32_t>((static_cast<unsigned long long>(n) * mul) >> 32) >> shift;
  }
};

struct PaArgs {
  const void* k;
  const void* v;
  long page_stride, row_stride, head_stride;
  int n_pages, hkv;
  FastDiv page_rows;
  const void* q;
  long ldq;
  void* out;
  long ldo;
  float* lse;
  int b, tq, hq;
  FastDiv group;      // G = hq / hkv
  FastDiv seq_rows;   // tq * G
  float scale;
  const int* prefix_pages;
  int prefix_len;
  const int* pages;
  int max_pages;
  int capacity;       // max_pages * page_rows
  const int* lens;
  // partial results: o [parts][b * tq * hq][hd], ml [parts][b * tq * hq]
  float* part_o;
  float2* part_ml;
  int parts;          // prefix splits, then own splits
  int prefix_splits, own_splits;
  int prefix_tiles, own_tiles;  // row tiles of a key head / of a (sequence, key head)
  int prefix_items;   // hkv * prefix_tiles * prefix_splits
  int* err;
};

// A block of rows against a range of one segment's keys.
struct PaItem {
  int seq;        // -1: the prefix
  int head;       // key head
  int row0;       // first of the tile's rows among the segment's
  int rows;       // the segment's rows
  int part;       // where its partial results go
  int k0, k1;     // keys
};

__device__ __forceinline__ int seq_len(const PaArgs& a, int s) {
  const int n = a.lens[s];
  if (n > a.capacity) {
    if (a.err) atomicExch(a.err, kErrIndex);
    return a.capacity;
  }
  return n;
}

// Token (sequence, query) and query head of row i of a segment.
struct PaRow {
  int s, t, h;
  long token;  // s * tq + t
};
__device__ __forceinline__ PaRow row_of(const PaArgs& a, const PaItem& w, int i) {
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

// How many of the segment's keys row r sees (a prefix of them).
__device__ __forceinline__ int visible(const PaArgs& a, bool prefix, const PaRow& r) {
  const int n = seq_len(a, r.s);
  if (n < 0) return 0;
  const int own = n - a.tq + r.t + 1;
  if (!prefix) return max(own, 0);
  return max(min(a.prefix_len + own, a.prefix_len), 0);
}

// Item `i` of the launch: the prefix's items, row tiles fastest (blocks that
// run together share keys), then the sequences' own.
__device__ __forceinline__ PaItem item_at(const PaArgs& a, int i, int tile_rows, int tile_keys) {
  PaItem w;
  int len, splits, split;
  if (i < a.prefix_items) {
    const int tile = i % a.prefix_tiles;
    i /= a.prefix_tiles;
    w.seq = -1;
    w.head = i % a.hkv;
    split = i / a.hkv;
    w.row0 = tile * tile_rows;
    w.rows = a.b * a.seq_rows.d;
    w.part = split;
    len = a.prefix_len;
    splits = a.prefix_splits;
  } else {
    i -= a.prefix_items;
    const int tile = i % a.own_tiles;
    i /= a.own_tiles;
    w.head = i % a.hkv;
    i /= a.hkv;
    w.seq = i / a.own_splits;
    split = i - w.seq * a.own_splits;
    w.row0 = tile * tile_rows;
    w.rows = a.seq_rows.d;
    w.part = a.prefix_splits + split;
    len = max(seq_len(a, w.seq), 0);
    splits = a.own_splits;
  }
  const int tiles = (len + tile_keys - 1) / tile_keys;
  w.k0 = static_cast<int>(static_cast<long>(tiles) * split / splits) * tile_keys;
  w.k1 = min(static_cast<int>(static_cast<long>(tiles) * (split + 1) / splits) * tile_keys, len);
  return w;
}

// Element offset of key j of the segment (head 0).
__device__ __forceinline__ long key_offset(const PaArgs& a, const int* table, int j) {
  const int p = a.page_rows(j);
  int page = table[p];
  if (page < 0 || page >= a.n_pages) {
    if (a.err) atomicExch(a.err, kErrIndex);
    page = 0;
  }
  return page * a.page_stride + static_cast<long>(j - p * a.page_rows.d) * a.row_stride;
}
__device__ __forceinline__ const int* table_of(const PaArgs& a, const PaItem& w) {
  return w.seq < 0 ? a.prefix_pages : a.pages + static_cast<long>(w.seq) * a.max_pages;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace sb
