// Attention over a paged key / value cache whose sequences share a prefix:
// dispatch, the CUDA-core kernel (float32), and the join of partial results.
#include <algorithm>

#include "prefix_attention.cuh"
#include "sb_kernels.h"
#define SB_PDL_FAMILY 2
#include "sb_launch.cuh"

namespace sb {

int num_sms_cached();
int warp_blocks_per_sm(int hd);

namespace {

constexpr int kRows = 16;  // rows of a block: 4 warps of 4
constexpr int kKeys = 32;  // keys of a tile: one a lane
constexpr int kThreads = 128;

template <int HD>
struct SimtShared {
  float q[kRows][HD];
  float k[2][kKeys][HD + 4];  // padded: the lanes of a warp read a row each
  float v[2][kKeys][HD];
  float p[kThreads / 32][kKeys][4];
};

// Scores, softmax and output of 16 rows against a range of keys, all in
// float32. A warp owns 4 rows: a lane computes the scores of its key with
// them, then the output columns lane * HD / 32 .. over the tile's keys.
template <int HD>
__device__ void attend_piece(const PaArgs& a, const PaPiece& w, SimtShared<HD>& sh) {
  using T = float;
  constexpr int C = HD / 32;  // output columns of a lane
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int* table = table_of(a, w);
  const bool prefix = w.seq < 0;

  PaRow row[4];
  int seen[4], most = 0, least = 0x7fffffff;  // keys that a row sees
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = w.row0 + warp * 4 + r;
    seen[r] = 0;
    if (i < w.rows) {
      row[r] = row_of(a, w, i);
      seen[r] = visible(a, prefix, row[r]);
      least = min(least, seen[r]);
    }
    most = max(most, seen[r]);
  }
  const int k1 = __syncthreads_or(most > w.k0) ? w.k1 : w.k0;  // shared memory is free, too
  const int warp_k1 = min(k1, most);

  for (int i = tid; i < kRows * HD; i += kThreads) {
    const int r = w.row0 + i / HD;
    float q = 0.f;
    if (r < w.rows) {
      const PaRow x = row_of(a, w, r);
      q = static_cast<float>(static_cast<const T*>(a.q)[x.token * a.ldq + static_cast<long>(x.h) * HD + i % HD]);
    }
    sh.q[i / HD][i % HD] = q;
  }

  const auto load = [&](int stage, int j0) {
    constexpr int V = 16 / sizeof(T), CH = HD / V;  // vectors of a row
    for (int i = tid; i < kKeys * CH; i += kThreads) {
      const int j = i / CH, c = i % CH * V;
      const bool in = j0 + j < k1;
      const long at = in ? key_offset(a, table, j0 + j) + w.head * a.head_stride + c : 0;
      const T* k = static_cast<const T*>(a.k) + at;
      const T* v = static_cast<const T*>(a.v) + at;
      cp_async16(smem_u32(&sh.k[stage][j][c]), k, in);
      cp_async16(smem_u32(&sh.v[stage][j][c]), v, in);
    }
    cp_async_commit();
  };

  float m[4], l[4], o[4][C];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) o[r][c] = 0.f;
  }
  if (w.k0 < k1) load(0, w.k0);
  int stage = 0;
  for (int j0 = w.k0; j0 < k1; j0 += kKeys, stage ^= 1) {
    if (j0 + kKeys < k1) {
      load(stage ^ 1, j0 + kKeys);
      cp_async_wait<1>();
    } else {
      cp_async_wait<0>();
    }
    __syncthreads();
    if (j0 < warp_k1) {
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
      for (int c = 0; c < HD; c += 4) {
        const float4 k = *reinterpret_cast<const float4*>(&sh.k[stage][lane][c]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float4 q = *reinterpret_cast<const float4*>(&sh.q[warp * 4 + r][c]);
          s[r] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, s[r]))));
        }
      }
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[r] = j0 + lane < seen[r] ? s[r] * a.scale : -INFINITY;
        float t = s[r];
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, x));
        const float mn = fmaxf(m[r], t);
        // a row that has seen no key keeps m = -inf, l = 0; NaN scores, which
        // the maximum passes over, go to p whatever it is
        const float f = mn == -INFINITY ? 1.f : expf(m[r] - mn);
        p[r] = expf(s[r] - (mn == -INFINITY ? 0.f : mn));
        l[r] = l[r] * f + p[r];
        m[r] = mn;
#pragma unroll
        for (int c = 0; c < C; ++c) o[r][c] *= f;
      }
      *reinterpret_cast<float4*>(&sh.p[warp][lane][0]) = make_float4(p[0], p[1], p[2], p[3]);
      __syncwarp();
      if (j0 + kKeys <= least) {
#pragma unroll 8
        for (int j = 0; j < kKeys; ++j) {
          const float4 q = *reinterpret_cast<const float4*>(&sh.p[warp][j][0]);
          float v[C];
#pragma unroll
          for (int c = 0; c < C; ++c) v[c] = sh.v[stage][j][lane * C + c];
#pragma unroll
          for (int c = 0; c < C; ++c) {
            o[0][c] = fmaf(q.x, v[c], o[0][c]);
            o[1][c] = fmaf(q.y, v[c], o[1][c]);
            o[2][c] = fmaf(q.z, v[c], o[2][c]);
            o[3][c] = fmaf(q.w, v[c], o[3][c]);
          }
        }
      } else {
        // some row stops inside the tile: a key that it does not see must
        // not reach it, whatever its values hold (0 * NaN)
        const int n = min(kKeys, warp_k1 - j0);
        for (int j = 0; j < n; ++j) {
          const float4 q = *reinterpret_cast<const float4*>(&sh.p[warp][j][0]);
          const float pr[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const float v = sh.v[stage][j][lane * C + c];
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (j0 + j < seen[r]) o[r][c] = fmaf(pr[r], v, o[r][c]);
          }
        }
      }
    }
    __syncthreads();
  }

#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (w.row0 + warp * 4 + r >= w.rows) continue;
    float sum = l[r];
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    const long at = row[r].token * a.hq + row[r].h;
    if (a.direct) {
      // (a row of zeros where nothing counts: o may hold 0 * inf)
      const float f = sum > 0.f ? 1.f / sum : sum;
      T* out = static_cast<T*>(a.out) + row[r].token * a.ldo + static_cast<long>(row[r].h) * HD + lane * C;
#pragma unroll
      for (int c = 0; c < C; ++c) out[c] = sum == 0.f ? T(0.f) : static_cast<T>(o[r][c] * f);
      if (a.lse && lane == 0) a.lse[at] = m[r] + logf(sum);
    } else {
      const long slot = static_cast<long>(w.part) * a.b * a.tq * a.hq + at;
      if (lane == 0) a.part_ml[slot] = make_float2(m[r], sum);
      if (sum != 0.f)
#pragma unroll
        for (int c = 0; c < C; ++c) a.part_o[slot * HD + lane * C + c] = o[r][c];
    }
  }
}

// The same for 64 rows, 16 a warp: a lane computes the scores of 4 rows with 4
// keys, then 4 rows of HD / 8 output columns, so that each 16 bytes read from
// shared memory serve 8 or more multiply-adds and these bound the kernel.
// (With 4 rows a warp the shared-memory reads do: 8 x 41 queries of 4 heads of
// 128 behind 10565 keys took 590 us; this takes 293, 24 TFLOP/s, with 8 warps
// an SM, too few to cover the latency of the arithmetic.)
constexpr int kWideRows = 64;

template <int HD>
struct WideShared {
  float q[kWideRows][HD + 4];
  float k[2][kKeys][HD + 4];
  float v[2][kKeys][HD];
  float p[kThreads / 32][kKeys][16];
};

template <int HD>
__device__ void attend_wide(const PaArgs& a, const PaPiece& w, WideShared<HD>& sh) {
  constexpr int Q = HD / 32;  // groups of 4 output columns a lane has
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int rg = lane / 8, kg = lane % 8;  // rows 4 rg .., keys kg + 8 i
  const int* table = table_of(a, w);

  PaRow row[4];
  int seen[4], most = 0, least = 0x7fffffff;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = w.row0 + warp * 16 + rg * 4 + r;
    seen[r] = w.k1;  // a row of no one sees all and is not stored
    if (i < w.rows) {
      row[r] = row_of(a, w, i);
      seen[r] = min(visible(a, w.seq < 0, row[r]), w.k1);
      most = max(most, seen[r]);
      if (seen[r] > w.k0) least = min(least, seen[r]);
    }
  }
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  const int k1 = __syncthreads_or(most > w.k0) ? w.k1 : w.k0;  // shared memory is free, too

  // Where no row sees a key of the piece nothing is copied: only the loop over
  // the keys waits for copies, and one still in flight behind it would meet
  // the next piece's in the same places, in no order.
  constexpr int CH = HD / 4;  // vectors of a row
  for (int i = w.k0 < k1 ? tid : kWideRows * CH; i < kWideRows * CH; i += kThreads) {
    const int r = w.row0 + i / CH, c = i % CH * 4;
    const bool in = r < w.rows;
    long at = 0;
    if (in) {
      const PaRow x = row_of(a, w, r);
      at = x.token * a.ldq + static_cast<long>(x.h) * HD + c;
    }
    cp_async16(smem_u32(&sh.q[i / CH][c]), static_cast<const float*>(a.q) + at, in);
  }
  const auto load = [&](int stage, int j0) {
#pragma unroll 4
    for (int i = tid; i < kKeys * CH; i += kThreads) {
      const int j = i / CH, c = i % CH * 4;
      const bool in = j0 + j < k1;
      const long at = in ? key_offset(a, table, j0 + j) + w.head * a.head_stride + c : 0;
      cp_async16(smem_u32(&sh.k[stage][j][c]), static_cast<const float*>(a.k) + at, in);
      cp_async16(smem_u32(&sh.v[stage][j][c]), static_cast<const float*>(a.v) + at, in);
    }
    cp_async_commit();
  };

  float m[4], l[4], o[4][Q][4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < Q; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[r][c][e] = 0.f;
  }
  if (w.k0 < k1) load(0, w.k0);
  int stage = 0;
  for (int j0 = w.k0; j0 < k1; j0 += kKeys, stage ^= 1) {
    if (j0 + kKeys < k1) {
      load(stage ^ 1, j0 + kKeys);
      cp_async_wait<1>();
    } else {
      cp_async_wait<0>();
    }
    __syncthreads();
    if (j0 < most) {
      float s[4][4] = {};  // row, key
#pragma unroll 4
      for (int c = 0; c < HD; c += 4) {
        float4 q[4], k[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) q[r] = *reinterpret_cast<const float4*>(&sh.q[warp * 16 + rg * 4 + r][c]);
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = *reinterpret_cast<const float4*>(&sh.k[stage][kg + 8 * i][c]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[r][i] = fmaf(q[r].x, k[i].x, fmaf(q[r].y, k[i].y, fmaf(q[r].z, k[i].z, fmaf(q[r].w, k[i].w, s[r][i]))));
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float t = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[r][i] = j0 + kg + 8 * i < seen[r] ? s[r][i] * a.scale : -INFINITY;
          t = fmaxf(t, s[r][i]);
        }
#pragma unroll
        for (int x = 4; x > 0; x >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, x));
        const float mn = fmaxf(m[r], t);
        const float f = mn == -INFINITY ? 1.f : expf(m[r] - mn);
        const float sub = mn == -INFINITY ? 0.f : mn;  // a NaN score stays one
        l[r] *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[r][i] = expf(s[r][i] - sub);
          l[r] += s[r][i];
        }
        m[r] = mn;
#pragma unroll
        for (int c = 0; c < Q; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[r][c][e] *= f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float4*>(&sh.p[warp][kg + 8 * i][rg * 4]) = make_float4(s[0][i], s[1][i], s[2][i], s[3][i]);
      __syncwarp();
      // where some row stops inside the tile, a key that it does not see must
      // not reach it, whatever its values hold (0 * NaN)
      const bool care = j0 + kKeys > least;
      const int n = min(kKeys, k1 - j0);
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const float4 p4 = *reinterpret_cast<const float4*>(&sh.p[warp][j][rg * 4]);
        const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
        for (int c = 0; c < Q; ++c) {
          const float4 v4 = *reinterpret_cast<const float4*>(&sh.v[stage][j][c * 32 + kg * 4]);
          const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (care && j0 + j >= seen[r]) continue;
              o[r][c][e] = fmaf(p[r], v[e], o[r][c][e]);
            }
        }
      }
    }
    __syncthreads();
  }

#pragma unroll
  for (int r = 0; r < 4; ++r) {
    float sum = l[r];
#pragma unroll
    for (int x = 4; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if (w.row0 + warp * 16 + rg * 4 + r >= w.rows) continue;
    const long at = row[r].token * a.hq + row[r].h;
    if (a.direct) {
      // (a row of zeros where nothing counts: o may hold 0 * inf)
      const float f = sum > 0.f ? 1.f / sum : sum;
      float* out = static_cast<float*>(a.out) + row[r].token * a.ldo + static_cast<long>(row[r].h) * HD + kg * 4;
#pragma unroll
      for (int c = 0; c < Q; ++c)
        *reinterpret_cast<float4*>(out + c * 32) =
            sum == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                       : make_float4(o[r][c][0] * f, o[r][c][1] * f, o[r][c][2] * f, o[r][c][3] * f);
      if (a.lse && kg == 0) a.lse[at] = m[r] + logf(sum);
    } else {
      const long slot = static_cast<long>(w.part) * a.b * a.tq * a.hq + at;
      if (kg == 0) a.part_ml[slot] = make_float2(m[r], sum);
      if (sum != 0.f)
#pragma unroll
        for (int c = 0; c < Q; ++c)
          *reinterpret_cast<float4*>(a.part_o + slot * HD + c * 32 + kg * 4) =
              make_float4(o[r][c][0], o[r][c][1], o[r][c][2], o[r][c][3]);
    }
  }
}

// Blocks [0, prefix blocks) take runs of the prefix, the others own pieces,
// with 16 or 64 rows a block as the segment's tiles have.
template <int HD>
__global__ void __launch_bounds__(kThreads) attn_simt_kernel(PaArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SimtShared<HD>& sh = *reinterpret_cast<SimtShared<HD>*>(smem_raw);
  WideShared<HD>& wide = *reinterpret_cast<WideShared<HD>*>(smem_raw);
  pdl_wait();
  pdl_trigger();
  const int cta = blockIdx.x;
  PaPiece w;
  if (cta < a.prefix.ctas) {
    PaRun run(a.prefix, a.hkv.d, cta);
    while (run.next(a, cta, w)) {
      if (a.prefix.tile_rows == kWideRows)
        attend_wide<HD>(a, w, wide);
      else
        attend_piece<HD>(a, w, sh);
    }
  } else {
    w = own_piece(a, cta - a.prefix.ctas);
    if (a.own.tile_rows == kWideRows)
      attend_wide<HD>(a, w, wide);
    else
      attend_piece<HD>(a, w, sh);
  }
}

// Joins a row's partial results with WPR warps, each taking every WPR-th part
// in order, then the warps in order. A part that saw no key (l = 0) left no
// output and is not read.
template <typename T, int HD, int WPR>
__global__ void __launch_bounds__(256) attn_join_kernel(PaArgs a) {
  constexpr int C = HD / 32;
  __shared__ float sh_o[WPR > 1 ? 8 : 1][HD];
  __shared__ float2 sh_ml[8];
  const long rows = static_cast<long>(a.b) * a.tq * a.hq;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long at = WPR == 1 ? static_cast<long>(blockIdx.x) * 8 + warp : blockIdx.x;
  const int first = WPR == 1 ? 0 : warp;
  pdl_wait();
  if (WPR == 1 && at >= rows) return;
  const long token = at / a.hq;
  const int h = static_cast<int>(at - token * a.hq);
  int n_prefix = 0;
  if (a.prefix.ctas > 0) {
    const int head = a.group(h);
    const long row = token * a.group.d + (h - head * static_cast<int>(a.group.d));
    n_prefix = a.prefix.parts_of(head * static_cast<int>(a.prefix.row_tiles.d) + static_cast<int>(row / a.prefix.tile_rows));
  }
  const int parts = n_prefix + a.own.parts;
  const auto slot = [&](int p) { return (p < n_prefix ? p : a.prefix.parts + p - n_prefix) * rows + at; };
  float m = -INFINITY, l = 0.f, o[C];
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] = 0.f;
  // groups of U parts: their loads are in flight together
  constexpr int U = 4;
  for (int p0 = first; p0 < parts; p0 += U * WPR) {
    float2 ml[U];
    float v[U][C];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int p = p0 + u * WPR;
      ml[u] = p < parts ? a.part_ml[slot(p)] : make_float2(-INFINITY, 0.f);
      const float* src = a.part_o + slot(min(p, parts - 1)) * HD + lane * C;
#pragma unroll
      for (int c = 0; c < C; ++c) v[u][c] = src[c];  // counts only where l is not 0
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (ml[u].y != 0.f) mn = fmaxf(mn, ml[u].x);
    const float f0 = l != 0.f ? expf(m - mn) : 0.f;
    l *= f0;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] *= f0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (ml[u].y == 0.f) continue;
      const float f = expf(ml[u].x - mn);
      l = fmaf(ml[u].y, f, l);
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] = fmaf(v[u][c], f, o[c]);
    }
    m = mn;
  }
  if (WPR > 1) {
#pragma unroll
    for (int c = 0; c < C; ++c) sh_o[warp][lane * C + c] = o[c];
    if (lane == 0) sh_ml[warp] = make_float2(m, l);
    __syncthreads();
    if (warp > 0) return;
    m = -INFINITY;
#pragma unroll
    for (int w = 0; w < WPR; ++w)
      if (sh_ml[w].y != 0.f) m = fmaxf(m, sh_ml[w].x);
    l = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = 0.f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) {
      if (sh_ml[w].y == 0.f) continue;
      const float f = expf(sh_ml[w].x - m);
      l = fmaf(sh_ml[w].y, f, l);
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] = fmaf(sh_o[w][lane * C + c], f, o[c]);
    }
  }
  const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  T* out = static_cast<T*>(a.out) + token * a.ldo + static_cast<long>(h) * HD + lane * C;
#pragma unroll
  for (int c = 0; c < C; ++c) out[c] = static_cast<T>(o[c] * f);
  if (a.lse && lane == 0) a.lse[at] = m + logf(l);
}

// Rows of the tiled copies that follow a page table: the largest power of two
// that divides a page, at most `most`; 0 where such a copy cannot (it would not
// start on the swizzle's 8 rows, or the strides are none that a tensor map
// takes).
int tiled_rows(const sb_kv_cache& c, int most) {
  const auto strides = [](int64_t s, int count) { return count == 1 || (s > 0 && s < (int64_t{1} << 38)); };
  if (c.page_rows % 8 || !strides(c.page_stride, c.n_pages) || !strides(c.row_stride, c.page_rows) ||
      !strides(c.head_stride, c.n_heads))
    return 0;
  return std::min(c.page_rows & -c.page_rows, most);
}

// Which kernel takes a segment, and how its keys are cut.
enum Kernel { kSimt, kWarp, kMma, kTc };
struct Plan {
  PaPrefix prefix = {};
  PaOwn own = {};
  Kernel prefix_kernel, own_kernel;
  int own_ctas = 0;
  long parts() const { return prefix.parts + own.parts; }
};

long ceil_div(long a, long b) { return (a + b - 1) / b; }

bool plan_of(const PrefixAttnDesc& d, Plan& p) {
  const long G = d.h_q / d.cache.n_heads, hkv = d.cache.n_heads;
  const long prefix_rows = static_cast<long>(d.b) * d.tq * G, own_rows = d.tq * G;
  // Up to 16 rows a warp each; tcgen05 tiles for more than 64, and from 17 on
  // where a hundred key tiles spread the start and end of its blocks: 32 rows of
  // 8 key heads behind 131072 keys 117 us, the warp-level kernel 147; behind
  // 8192, 27 and 32; 64 rows behind 8192, 28 and 41; behind 1024 the same.
  const auto choose = [&](long rows, long items, long keys) {
    if (d.cache.elem == SB_ELEM_F32) return kSimt;
    if (rows <= 16) return kWarp;
    if (d.cache.n_pages == 0 || !tiled_rows(d.cache, 128)) return kMma;  // (no tensor map of no memory)
    return rows > 64 || items * (keys / 128) >= 100L ? kTc : kMma;
  };
  const auto rows_of = [](Kernel k, long rows) {
    if (k == kTc) return rows > 128 ? 256 : 128;
    if (k == kSimt) return rows <= 16 ? kRows : kWideRows;
    return k == kWarp ? 16 : (rows <= 32 ? 32 : 64);
  };
  const auto keys_of = [](Kernel k) { return k == kTc ? 128 : (k == kMma ? 64 : (k == kWarp ? 16 : kKeys)); };
  const long own_capacity = static_cast<long>(d.max_pages) * d.cache.page_rows;
  p.prefix_kernel = choose(prefix_rows, hkv, d.prefix_len);
  p.own_kernel = choose(own_rows, d.b * hkv, own_capacity);
  p.prefix.tile_rows = rows_of(p.prefix_kernel, prefix_rows);
  p.own.tile_rows = rows_of(p.own_kernel, own_rows);
  p.prefix.tile_keys = keys_of(p.prefix_kernel);
  p.own.tile_keys = keys_of(p.own_kernel);
  const long prefix_row_tiles = ceil_div(prefix_rows, p.prefix.tile_rows);
  const long own_row_tiles = ceil_div(own_rows, p.own.tile_rows);
  const long own_tiles = ceil_div(own_capacity, p.own.tile_keys);
  long prefix_tiles = ceil_div(d.prefix_len, p.prefix.tile_keys);
  long prefix_work = hkv * prefix_row_tiles * prefix_tiles;
  const long own_items = d.b * hkv * own_row_tiles, own_work = own_items * own_tiles;
  // Key tiles that a block takes: at least 2, and enough that all blocks of a
  // launch are resident at once.
  const bool together = p.prefix_kernel == p.own_kernel;
  const auto quota = [&](Kernel k, long work) {
    const long blocks = k == kTc ? 1 : (k == kWarp ? warp_blocks_per_sm(d.cache.head_dim) : 2);
    return std::max(k == kWarp ? 4L : 2L, ceil_div(work, blocks * num_sms_cached()));
  };
  const long own_quota = quota(p.own_kernel, own_work + (together ? prefix_work : 0));
  long prefix_quota = quota(p.prefix_kernel, prefix_work + (together ? own_work : 0));
  if (p.prefix_kernel == kTc && prefix_work > 0 && !together) {
    long sms = num_sms_cached();
    // Own keys of one-warp blocks run beside the prefix: a tcgen05 block costs
    // about 10 us beyond its key tiles, so it takes more of them on fewer SMs,
    // and the own keys' blocks fill the others and, as they come free, these.
    // A 256-row tile costs an SM as much as 7 of the warps' 16-key tiles; about
    // a third of the own capacity is counted, since lengths are on the device
    // and too many SMs cost less than too few. That suits lengths spread over
    // the capacity (64 x 32 queries behind 8192 and 0..512 own keys 39 us, in a
    // row of calls) as well as equal ones below it (256 each: 40, 8 each: 38);
    // with the capacity full the own keys end last (512 each: 51). Against one
    // block an SM, other work between the calls: 49 -> 41 us, counting a sixth
    // 48; 100 of them behind 20000, 96 -> 73. Beyond 24 tiles, or an eighth more than all
    // SMs would give, nothing is gained (512 behind 16384 and up to 256: 201 at
    // half as many again, 198 here), and the prefix could end last (512 behind
    // 400 and up to 600: 136 us, 282 without this limit).
    if (p.own_kernel == kWarp && own_work > 0) {
      const long own = own_work * 256 / p.prefix.tile_rows / 20;
      sms = std::max(1L, sms * prefix_work / (prefix_work + own));
      prefix_quota = std::min(std::max(2L, ceil_div(prefix_work, sms)), std::max(24L, prefix_quota * 9 / 8));
      sms = std::max(sms, ceil_div(prefix_work, prefix_quota));
    }
    // Runs that end with an item, where they are not much longer: a second
    // piece costs a block 2.5 tiles (64 queries as above, 8 tiles a block 45
    // us, 7 and 9: 49 and 50; 512 and next to no own keys, 64 tiles 135, 56:
    // 140, under the power cap 151 and 158).
    const long each = sms / (hkv * prefix_row_tiles);  // blocks an item
    if (each > 0) {
      const long even = std::max(2L, ceil_div(prefix_tiles, each));
      if (8 * even <= 9 * prefix_quota + 20) {
        prefix_quota = even;
        prefix_tiles = ceil_div(prefix_tiles, even) * even;
        prefix_work = hkv * prefix_row_tiles * prefix_tiles;
      }
    }
  }
  if (prefix_work + prefix_quota > 0x7fffffffL) return false;  // counted in 32 bits
  p.prefix.row_tiles = FastDiv::of(static_cast<uint32_t>(prefix_row_tiles));
  p.prefix.tiles = FastDiv::of(static_cast<uint32_t>(std::max(1L, prefix_tiles)));
  p.prefix.per_cta = FastDiv::of(static_cast<uint32_t>(prefix_quota));
  p.prefix.ctas = static_cast<int>(ceil_div(prefix_work, prefix_quota));
  long splits = std::min(256L, ceil_div(own_tiles, own_quota));
  if (prefix_work + splits == 0) splits = 1;  // no keys at all: an empty part
  // a block of the tcgen05 kernel with one row tile deals its key tiles, where
  // it has several, out to both of its softmax groups
  p.prefix.slots = p.prefix_kernel == kTc && p.prefix.tile_rows == 128 && prefix_tiles > 1 ? 2 : 1;
  p.own.slots = p.own_kernel == kTc && p.own.tile_rows == 128 && own_tiles >= 2 * splits ? 2 : 1;
  p.prefix.parts = prefix_work ? static_cast<int>((prefix_tiles - 1) / prefix_quota + 2) : 0;
  if (prefix_work && prefix_quota % prefix_tiles == 0) p.prefix.parts = 1;  // whole items a block
  if (prefix_work && prefix_tiles % prefix_quota == 0) p.prefix.parts = static_cast<int>(prefix_tiles / prefix_quota);
  p.prefix.parts *= p.prefix.slots;
  p.own.row_tiles = FastDiv::of(static_cast<uint32_t>(own_row_tiles));
  p.own.splits = FastDiv::of(static_cast<uint32_t>(std::max(1L, splits)));
  p.own.parts = static_cast<int>(splits) * p.own.slots;
  const long own_ctas = own_items * splits;
  if (own_ctas + p.prefix.ctas > 0x7fffffffL) return false;
  p.own_ctas = static_cast<int>(own_ctas);
  return true;
}

}  // namespace

// Tensor map over the pages of k or v: [page][row][head][head_dim], boxes of
// 64 values of a head in box_rows rows.
bool cache_map(void* map, const void* base, const PaArgs& a, int hd) {
  const long dims[4] = {hd, static_cast<long>(a.hkv.d), static_cast<long>(a.page_rows.d), a.n_pages};
  // the stride of a dimension of one is free, but the map wants a usable one
  const auto bytes = [&](long s, long count) { return count == 1 ? 16 * 16 : s * 2; };
  const long strides[3] = {bytes(a.head_stride, dims[1]), bytes(a.row_stride, dims[2]), bytes(a.page_stride, dims[3])};
  return make_tma_4d_bf16(map, base, dims, strides, 64, a.box_rows);
}

namespace {

template <int HD>
int simt(const PaArgs& a, int own_ctas, cudaStream_t s) {
  const bool wide = (a.prefix.ctas > 0 && a.prefix.tile_rows == kWideRows) || (own_ctas > 0 && a.own.tile_rows == kWideRows);
  const size_t smem = wide ? sizeof(WideShared<HD>) : sizeof(SimtShared<HD>);
  static bool attr = false;
  if (!attr) {
    if (cudaFuncSetAttribute(attn_simt_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(std::max(sizeof(WideShared<HD>), sizeof(SimtShared<HD>)))) != cudaSuccess)
      return SB_OPERR_LAUNCH;
    attr = true;
  }
  return launch_pdl(attn_simt_kernel<HD>, dim3(static_cast<unsigned>(a.prefix.ctas) + own_ctas), dim3(kThreads), smem,
                    s, a) == cudaSuccess
             ? 0
             : SB_OPERR_LAUNCH;
}

template <typename T, int HD>
int join(const PaArgs& a, cudaStream_t s) {
  const long rows = static_cast<long>(a.b) * a.tq * a.hq;
  const bool wide = a.prefix.parts + a.own.parts > 8;
  const dim3 grid(static_cast<unsigned>(wide ? rows : (rows + 7) / 8));
  return launch_pdl(wide ? attn_join_kernel<T, HD, 8> : attn_join_kernel<T, HD, 1>, grid, dim3(256), 0, s, a) ==
                 cudaSuccess
             ? 0
             : SB_OPERR_LAUNCH;
}
template <typename T>
int join(const PaArgs& a, int hd, cudaStream_t s) {
  return hd == 32 ? join<T, 32>(a, s) : (hd == 64 ? join<T, 64>(a, s) : join<T, 128>(a, s));
}

size_t align16(size_t n) { return (n + 15) & ~size_t{15}; }

}  // namespace

// `early`: a kernel that starts beside the one before it on the stream, which
// writes nothing that it reads or writes and whose blocks all have started, so
// its own predecessors have completed. One block waits for that kernel at its
// end: whoever waits for the second then has the first's results as well.
int attn_mma(const PaArgs& a, int hd, int prefix_ctas, int own_ctas, bool early, cudaStream_t s);
int attn_warp(const PaArgs& a, int hd, int prefix_ctas, int own_ctas, bool early, cudaStream_t s);
int attn_tc(const PaArgs& a, int hd, int prefix_ctas, int own_ctas, bool early, cudaStream_t s);

size_t prefix_attention_workspace_bytes(const PrefixAttnDesc& d) {
  Plan p;
  if (d.b == 0 || d.tq == 0 || !plan_of(d, p) || p.parts() <= 1) return 0;
  const size_t rows = static_cast<size_t>(d.b) * d.tq * d.h_q;
  return align16(p.parts() * rows * sizeof(float2)) + p.parts() * rows * d.cache.head_dim * sizeof(float);
}

int prefix_attention(const PrefixAttnDesc& d, void* ws, size_t, cudaStream_t s, int* err) {
  Plan p;
  if (!plan_of(d, p)) return SB_OPERR_ARGS;
  PaArgs a = {};
  a.k = d.cache.k;
  a.v = d.cache.v;
  a.page_stride = d.cache.page_stride;
  a.row_stride = d.cache.row_stride;
  a.head_stride = d.cache.head_stride;
  a.n_pages = d.cache.n_pages;
  a.hkv = FastDiv::of(d.cache.n_heads);
  a.page_rows = FastDiv::of(d.cache.page_rows);
  a.q = d.q;
  a.ldq = d.ldq;
  a.out = d.out;
  a.ldo = d.ldo;
  a.lse = d.lse;
  a.b = d.b;
  a.tq = d.tq;
  a.hq = d.h_q;
  a.group = FastDiv::of(d.h_q / d.cache.n_heads);
  a.seq_rows = FastDiv::of(d.tq * (d.h_q / d.cache.n_heads));
  a.scale = d.scale;
  a.prefix_pages = d.prefix_pages;
  a.prefix_len = d.prefix_len;
  a.pages = d.pages;
  a.max_pages = d.max_pages;
  a.capacity = d.max_pages * d.cache.page_rows;
  a.lens = d.lens;
  a.prefix = p.prefix;
  a.own = p.own;
  a.direct = p.parts() == 1;
  a.box_rows = tiled_rows(d.cache, 128);
  const size_t rows = static_cast<size_t>(d.b) * d.tq * d.h_q;
  a.part_ml = static_cast<float2*>(ws);
  a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + align16(p.parts() * rows * sizeof(float2)));
  a.err = err;
  const int hd = d.cache.head_dim;
  const bool f32 = d.cache.elem == SB_ELEM_F32;
  int rc = 0;
  if (!f32) {
    // One launch for both segments, or the own keys' beside the prefix's: their
    // parts are apart, so the second starts once all blocks of the first have.
    const auto attend = [&](Kernel k, int prefix, int own, bool early) {
      if (prefix + own == 0) return 0;
      return (k == kTc ? attn_tc : (k == kMma ? attn_mma : attn_warp))(a, hd, prefix, own, early, s);
    };
    const bool together = p.prefix_kernel == p.own_kernel;
    rc = attend(p.prefix_kernel, a.prefix.ctas, together ? p.own_ctas : 0, false);
    if (!rc && !together) rc = attend(p.own_kernel, 0, p.own_ctas, a.prefix.ctas > 0);
  } else
    rc = hd == 32 ? simt<32>(a, p.own_ctas, s) : (hd == 64 ? simt<64>(a, p.own_ctas, s) : simt<128>(a, p.own_ctas, s));
  if (rc || a.direct) return rc;
  return f32 ? join<float>(a, hd, s) : join<__nv_bfloat16>(a, hd, s);
}

}  // namespace sb
