// Attention over a paged cache with a shared prefix, few rows a key head
// (bf16): reading the keys bounds it, so the kernels are built around rings of
// asynchronous copies, which follow pages of any size, and the products run as
// warp-level m16n8k16 matrix instructions on 16 rows, which take a fraction of
// the copies' time. (The tcgen05 kernel's tiles of 128 rows serve larger row
// blocks.) Up to 16 rows a warp works alone (second half of the file; own keys
// of 512 sequences of up to 256, 268 MB: 61 us, 0.67 of the measured copy rate,
// the latency of a warp's own instructions against 8 warps an SM); more rows
// that the tcgen05 kernel does not take:
//
// A block of 4 warps takes 32 or 64 rows against tiles of 64 keys: with 32 rows
// two warps share the keys of 16 rows, with 64 rows a warp has all keys of its
// 16. Warps that share rows keep their own maxima, sums and outputs and are
// joined once at the end through shared memory.
//
// Per 16 keys: s = q k^T in float32; the reference r of a row's exponents
// 2^(s - r) rises only when some score passes it by 8, so the output is
// rescaled rarely and p stays below 2^8; l sums p in float32; p is rounded
// to bf16 for the product with v, which accumulates in float32.
#include <algorithm>

#include "prefix_attention.cuh"
#include "sb_kernels.h"
#define SB_PDL_FAMILY 2
#include "sb_launch.cuh"

namespace sb {

int num_sms_cached();
constexpr int kWarpStages = 3;
constexpr int kWarpStageBytes = kWarpStages * 2 * 16 * 2;  // of its ring, per value of a head
// Blocks of the one-warp kernel that shared memory lets an SM hold (228 KB,
// 1 KB a block to the system; at most 16, which keep enough in flight).
int warp_blocks_per_sm(int hd) { return std::min(16, 228 * 1024 / (kWarpStageBytes * hd + 12 * hd + 1024)); }

namespace {

constexpr int kKeys = 64;
constexpr int kThreads = 128;

template <int HD>
struct MmaShared {
  static constexpr int kStages = HD == 128 ? 3 : 4;
  static constexpr int kTile = kKeys * HD;  // values
  __nv_bfloat16 kv[kStages][2][kTile];
  long offset[2][kKeys];  // of the keys of the next tiles to load
  int bad[3 * HD];        // first key with NaN, +inf, -inf in a column of v
  int care;               // from this key on some row stops inside a tile
};

// 16-byte chunk c of row r of a tile, spread over the banks so that 8
// consecutive rows of one chunk are 8 different 16-byte columns.
template <int HD>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  constexpr int CH = HD / 8;  // chunks of a row
  const int x = HD >= 64 ? (r & 7) : ((r >> 1) & 3);
  return (r * CH + (c ^ x)) * 16;
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Takes NaN and infinities out of a tile of v (rows j0 .. of the segment),
// thread `tid` of N, and remembers the first key that has one in a column
// (bad: [NaN, +inf, -inf][HD]).
template <int HD, int KEYS, int N>
__device__ void clean_tile(__nv_bfloat16* tile, int* bad, int j0, int tid) {
  for (int i = tid; i < KEYS * HD / 8; i += N) {
    const int r = i / (HD / 8), c = i % (HD / 8);
    uint4* p = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(tile) + chunk_at<HD>(r, c));
    const uint4 u = *p;
    uint32_t w[4] = {u.x, u.y, u.z, u.w};
    bool any = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t b = (w[e / 2] >> (16 * (e % 2))) & 0xffffu;
      if ((b & 0x7f80u) != 0x7f80u) continue;
      any = true;
      w[e / 2] &= e % 2 ? 0x0000ffffu : 0xffff0000u;
      atomicMin(&bad[((b & 0x7fu) ? 0 : (b >> 15 ? 2 : 1)) * HD + c * 8 + e], j0 + r);
    }
    if (any) *p = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// What the values taken out of column c add to a row that sees `seen` keys.
template <int HD>
__device__ __forceinline__ float taken_out(const int* bad, int c, int seen) {
  const bool up = bad[HD + c] < seen, down = bad[2 * HD + c] < seen;
  if (bad[c] < seen || (up && down)) return __int_as_float(0x7fffffff);
  return up ? INFINITY : (down ? -INFINITY : 0.f);
}

// The state of 16 rows in one warp: lane l holds rows l / 4 and l / 4 + 8,
// columns (l % 4) * 2 and the next of each group of 8.
template <int HD>
struct Rows {
  static constexpr int KS = HD / 16;  // steps of 16 along head_dim
  uint32_t q[KS][4];
  int seen[2];   // keys of the segment that the rows see, at most the piece's end
  int lo;        // of the warp's rows, for masking
  float o[HD / 8][4];
  float ref[2], l[2];
  float lim[2];  // scores above it raise the reference; -inf where a row's is far out

  __device__ __forceinline__ void start(const PaArgs& a, const PaPiece& w, int row0) {
    const int g = threadIdx.x % 32 / 4, t4 = threadIdx.x % 4;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = row0 + g + 8 * r;
      seen[r] = w.k1;  // a row of no one sees all and is not stored
      if (i < w.rows) {
        const PaRow row = row_of(a, w, i);
        seen[r] = min(visible(a, w.seq < 0, row), w.k1);
        const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(a.q) + row.token * a.ldq +
                                 static_cast<long>(row.h) * HD + t4 * 2;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          q[s][r] = *reinterpret_cast<const uint32_t*>(p + s * 16);
          q[s][r + 2] = *reinterpret_cast<const uint32_t*>(p + s * 16 + 8);
        }
      } else {
#pragma unroll
        for (int s = 0; s < KS; ++s) q[s][r] = q[s][r + 2] = 0u;
      }
      ref[r] = lim[r] = -INFINITY;
      l[r] = 0.f;
    }
    lo = __reduce_min_sync(0xffffffffu, min(seen[0], seen[1]));
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  }

  // From this key on some row stops before the piece does. Such a row must
  // not meet the values behind its last key, even as 0 * NaN, so the tiles of
  // v from there on get their NaN and infinities taken out, to be added to
  // the rows that see them at the end. (A row that sees no key of the piece
  // is dropped by its l = 0.)
  __device__ __forceinline__ int care(const PaPiece& w) const {
    return __reduce_min_sync(0xffffffffu,
                             min(seen[0] > w.k0 ? seen[0] : w.k1, seen[1] > w.k0 ? seen[1] : w.k1));
  }

  // 16 keys, number key0 of the segment on, in rows r0 .. of the tiles sk, sv.
  __device__ __forceinline__ void take(uint32_t sk, uint32_t sv, int r0, int key0, float sl) {
    const int lane = threadIdx.x % 32, t4 = lane % 4;
    float s[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      // matrices: keys 0-7 and 8-15, each at head_dim 0-7 and 8-15 of the step
      uint32_t kb[4];
      ldmatrix4(kb, sk + chunk_at<HD>(r0 + (lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)));
      mma16816(s[0], q[ks], kb[0], kb[1]);
      mma16816(s[1], q[ks], kb[2], kb[3]);
    }
    if (key0 + 16 > lo) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (key0 + n * 8 + t4 * 2 + (e & 1) >= seen[e >> 1]) s[n][e] = -INFINITY;
    }
    float mx[2];
#pragma unroll
    for (int r = 0; r < 2; ++r)
      mx[r] = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1])) * sl;
    float by = sl;
    if (__any_sync(0xffffffffu, mx[0] > lim[0] || mx[1] > lim[1])) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        const float to = fmaxf(ref[r], mx[r]);
        const float f = to == -INFINITY ? 1.f : ex2_approx(ref[r] - to);
        ref[r] = to;
        l[r] *= f;
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) {
          o[n][2 * r] *= f;
          o[n][2 * r + 1] *= f;
        }
      }
      const bool far = __any_sync(0xffffffffu, far_out(ref[0]) || far_out(ref[1]));
      lim[0] = far ? -INFINITY : ref[0] + 8.f;
      lim[1] = far ? -INFINITY : ref[1] + 8.f;
      if (far) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[0][e] *= sl;
          s[1][e] *= sl;
        }
        by = 1.f;
      }
    }
    // p as the sum of two bf16: rounding it to one would add as much error as
    // the output's own rounding, and the second product is free beside the
    // reading of v
    uint32_t hi[4], rest[4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float sub = ref[r] == -INFINITY ? 0.f : ref[r];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float p0 = ex2_approx(fmaf(s[n][2 * r], by, -sub)), p1 = ex2_approx(fmaf(s[n][2 * r + 1], by, -sub));
        l[r] += p0 + p1;
        const uint32_t h = pack_bf16x2(p0, p1);
        hi[r + 2 * n] = h;
        rest[r + 2 * n] = pack_bf16x2(p0 - __uint_as_float(h << 16), p1 - __uint_as_float(h & 0xffff0000u));
      }
    }
#pragma unroll
    for (int n = 0; n < KS; ++n) {
      // matrices: keys 0-7 and 8-15 at columns 0-7, then at columns 8-15
      uint32_t vb[4];
      ldmatrix4_t(vb, sv + chunk_at<HD>(r0 + (lane & 15), n * 2 + (lane >> 4)));
      mma16816(o[2 * n], hi, vb[0], vb[1]);
      mma16816(o[2 * n + 1], hi, vb[2], vb[3]);
      mma16816(o[2 * n], rest, vb[0], vb[1]);
      mma16816(o[2 * n + 1], rest, vb[2], vb[3]);
    }
  }

  // A row's sum over the four lanes that hold its columns.
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
  }
};

template <int HD>
__device__ void attend_piece(const PaArgs& a, const PaPiece& w, int tile_rows, MmaShared<HD>& sh) {
  constexpr int CH = HD / 8;
  using SH = MmaShared<HD>;
  constexpr int ST = SH::kStages;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int wm = tile_rows / 16;       // warps along the rows
  const int mrow = (warp % wm) * 16;   // this warp's 16 rows of the tile
  const int kgroup = warp / wm;        // its share of a tile's keys: wm groups of 16
  const int* table = table_of(a, w);
  using bf = __nv_bfloat16;
  const bf* gk = static_cast<const bf*>(a.k) + static_cast<long>(w.head) * a.head_stride;
  const bf* gv = static_cast<const bf*>(a.v) + static_cast<long>(w.head) * a.head_stride;
  const float sl = a.scale * 1.4426950408889634f;

  // offsets of a tile's keys, computed a tile ahead of its loads
  const auto locate = [&](int slot, int j0) {
    if (tid < kKeys && j0 + tid < w.k1) sh.offset[slot][tid] = key_offset(a, table, j0 + tid);
  };
  const auto load = [&](int stage, int slot, int j0) {
    if (j0 < w.k1) {
#pragma unroll
      for (int i = 0; i < kKeys * CH / kThreads; ++i) {
        const int at = i * kThreads + tid, r = at / CH, c = at % CH;
        const bool in = j0 + r < w.k1;
        const long off = in ? sh.offset[slot][r] + c * 8 : 0;
        const uint32_t d = chunk_at<HD>(r, c);
        cp_async16(smem_u32(&sh.kv[stage][0][0]) + d, gk + off, in);
        cp_async16(smem_u32(&sh.kv[stage][1][0]) + d, gv + off, in);
      }
    }
    cp_async_commit();
  };

  __syncthreads();  // shared memory may still be read for the piece before
  for (int i = tid; i < 3 * HD; i += kThreads) sh.bad[i] = 0x7fffffff;
  if (tid == 0) sh.care = w.k1;
  locate(0, w.k0);
  __syncthreads();
  int slot = 0;
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) {
    load(s, slot, w.k0 + s * kKeys);
    locate(slot ^ 1, w.k0 + (s + 1) * kKeys);
    slot ^= 1;
    if (s + 1 < ST - 1) __syncthreads();
  }
  Rows<HD> rows;
  rows.start(a, w, w.row0 + mrow);
  const int lo = rows.care(w);
  if (lane == 0 && lo < w.k1) atomicMin(&sh.care, lo);

  int stage = 0;
  for (int j0 = w.k0; j0 < w.k1; j0 += kKeys) {
    cp_async_wait<ST - 2>();
    __syncthreads();
    {
      // the stage that this tile's predecessor used is free again
      const int ahead = j0 + (ST - 1) * kKeys;
      load(stage == 0 ? ST - 1 : stage - 1, slot, ahead);
      locate(slot ^ 1, ahead + kKeys);
      slot ^= 1;
    }
    const uint32_t sk = smem_u32(&sh.kv[stage][0][0]), sv = smem_u32(&sh.kv[stage][1][0]);
    const int end = min(j0 + kKeys, w.k1);
    if (sh.care < end) {
      clean_tile<HD, kKeys, kThreads>(&sh.kv[stage][1][0], sh.bad, j0, tid);
      __syncthreads();
    }
    for (int kg = kgroup * wm; kg < kgroup * wm + wm; ++kg) {
      if (j0 + kg * 16 >= end) break;
      rows.take(sk, sv, kg * 16, j0 + kg * 16, sl);
    }
    stage = stage == ST - 1 ? 0 : stage + 1;
  }
  cp_async_wait<0>();
  rows.finish();
  __syncthreads();  // the ring is free

  // join the warps that share rows, in the order of their keys
  const int wk = 4 / wm;  // 1 or 2
  constexpr int P = HD + 4;  // padded row of outputs
  float* buf = reinterpret_cast<float*>(&sh.kv[0][0][0]);  // [kgroup][tile_rows][P]: 64 rows at most
  float2* stat = reinterpret_cast<float2*>(buf + 64 * P);  // [kgroup][tile_rows]
  static_assert(64 * P * 4 + 64 * 8 <= sizeof(sh.kv), "the ring holds the outputs");
  const int g = lane / 4, t4 = lane % 4;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int at = kgroup * tile_rows + mrow + g + 8 * r;
    if (t4 == 0) stat[at] = make_float2(rows.ref[r], rows.l[r]);
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
      *reinterpret_cast<float2*>(&buf[at * P + n * 8 + t4 * 2]) = make_float2(rows.o[n][2 * r], rows.o[n][2 * r + 1]);
  }
  __syncthreads();
  // 4 columns a thread, HD / 4 threads a row
  constexpr int TPR = HD / 4;
  for (int i = tid / TPR; i < tile_rows; i += kThreads / TPR) {
    if (w.row0 + i >= w.rows) break;
    const PaRow x = row_of(a, w, w.row0 + i);
    const int c = tid % TPR * 4;
    float m = -INFINITY, sum = 0.f;
    for (int k = 0; k < wk; ++k) m = fmaxf(m, stat[k * tile_rows + i].x);
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < wk; ++k) {
      const float2 st = stat[k * tile_rows + i];
      if (st.y == 0.f) continue;
      const float f = ex2_approx(st.x - m);
      sum = fmaf(st.y, f, sum);
      const float4 u = *reinterpret_cast<const float4*>(&buf[(k * tile_rows + i) * P + c]);
      v[0] = fmaf(u.x, f, v[0]);
      v[1] = fmaf(u.y, f, v[1]);
      v[2] = fmaf(u.z, f, v[2]);
      v[3] = fmaf(u.w, f, v[3]);
    }
    if (sum != 0.f) {
      const int n = min(visible(a, w.seq < 0, x), w.k1);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += taken_out<HD>(sh.bad, c + e, n);
    }
    const float nat = m * 0.6931471805599453f;  // natural units outside
    const long at = x.token * a.hq + x.h;
    if (a.direct) {
      const float f = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
      *reinterpret_cast<uint2*>(static_cast<bf*>(a.out) + x.token * a.ldo + static_cast<long>(x.h) * HD + c) =
          make_uint2(pack_bf16x2(v[0] * f, v[1] * f), pack_bf16x2(v[2] * f, v[3] * f));
      if (a.lse && c == 0) a.lse[at] = nat + logf(sum);
    } else {
      const long slot_at = static_cast<long>(w.part) * a.b * a.tq * a.hq + at;
      if (c == 0) a.part_ml[slot_at] = make_float2(nat, sum);
      if (sum != 0.f) *reinterpret_cast<float4*>(a.part_o + slot_at * HD + c) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
}

// Blocks [0, prefix blocks) take runs of the prefix, the others own pieces.
// `early`: see attn_mma's declaration.
template <int HD>
__global__ void __launch_bounds__(kThreads, HD == 128 ? 2 : 3) attn_mma_kernel(PaArgs a, int prefix_ctas, int early) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  MmaShared<HD>& sh = *reinterpret_cast<MmaShared<HD>*>(smem_raw);
  if (!early) pdl_wait();
  pdl_trigger();
  const int cta = blockIdx.x;
  if (cta < prefix_ctas) {
    PaRun run(a.prefix, a.hkv.d, cta);
    PaPiece w;
    while (run.next(a, cta, w)) attend_piece<HD>(a, w, a.prefix.tile_rows, sh);
  } else {
    attend_piece<HD>(a, own_piece(a, cta - prefix_ctas), a.own.tile_rows, sh);
  }
  if (early && cta == 0) pdl_wait();
}

// ---- one warp a piece: at most 16 rows -------------------------------------
// A block is one warp with a ring of its own, 16 keys a stage, so blocks never
// wait for one another and as many as registers and shared memory hold (8 with
// 128 values a head) keep the SM's copies in flight. A block takes a run of the
// prefix or one own piece. (As many blocks as are resident, each taking every
// so-manyth own piece, left SMs idle a quarter of the time: 512 sequences of up
// to 256 keys took 72 us, a block each 62.)
template <int HD>
struct WarpShared {
  __nv_bfloat16 kv[kWarpStages][2][16 * HD];
  int bad[3 * HD];
};

struct WarpWork {
  PaRun run;
  int own;  // the own piece, or -1
  __device__ __forceinline__ WarpWork(const PaArgs& a, int prefix_ctas)
      : run(a.prefix, a.hkv.d, blockIdx.x), own(static_cast<int>(blockIdx.x) - prefix_ctas) {
    if (own >= 0) run.left = 0;
  }
  __device__ __forceinline__ bool next(const PaArgs& a, PaPiece& w) {
    if (own < 0) return run.next(a, blockIdx.x, w);
    w = own_piece(a, own);
    own = -1;
    return true;
  }
};

template <int HD>
__global__ void __launch_bounds__(32) attn_warp_kernel(PaArgs a, int prefix_ctas, int early) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  WarpShared<HD>& sh = *reinterpret_cast<WarpShared<HD>*>(smem_raw);
  using bf = __nv_bfloat16;
  constexpr int CH = HD / 8, ST = kWarpStages;
  const int lane = threadIdx.x;
  const float sl = a.scale * 1.4426950408889634f;
  if (!early) pdl_wait();
  pdl_trigger();

  // the copies' place in the work, ahead of the products'
  WarpWork ahead(a, prefix_ctas);
  PaPiece lw;
  lw.k1 = 0;
  int lj = 0;
  long off = 0;  // of key lj + lane % 16
  bool more = true;
  // One block reads a key, and the prefix's, which many read, stay in L2 (64
  // sequences beside a tcgen05 prefix of 8192 keys 44 -> 41 us).
  const uint64_t once = read_once_policy();
  const auto locate = [&] {
    const int j = lj + (lane & 15);
    off = j < lw.k1 ? key_offset(a, table_of(a, lw), j) + static_cast<long>(lw.head) * a.head_stride : 0;
  };
  const auto issue = [&](int stage) {
    while (more && lj >= lw.k1) {
      more = ahead.next(a, lw);
      if (!more) break;
      lj = lw.k0;
      if (lj < lw.k1) locate();
    }
    if (more) {
      const uint32_t sk = smem_u32(&sh.kv[stage][0][0]), sv = smem_u32(&sh.kv[stage][1][0]);
#pragma unroll
      for (int i = 0; i < 16 * CH / 32; ++i) {
        const int r = (i * 32 + lane) / CH, c = lane % CH;
        const long o = __shfl_sync(0xffffffffu, off, r) + c * 8;
        const bool in = lj + r < lw.k1;
        const uint32_t d = chunk_at<HD>(r, c);
        cp_async16(sk + d, static_cast<const bf*>(a.k) + (in ? o : 0), in, once);
        cp_async16(sv + d, static_cast<const bf*>(a.v) + (in ? o : 0), in, once);
      }
      lj += 16;
      if (lj < lw.k1) locate();
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) issue(s);

  WarpWork work(a, prefix_ctas);
  PaPiece w;
  int stage = 0;
  while (work.next(a, w)) {
    Rows<HD> rows;
    rows.start(a, w, w.row0);
    const int care = rows.care(w);
    const bool careful = care < w.k1;
    if (careful) {
      for (int i = lane; i < 3 * HD; i += 32) sh.bad[i] = 0x7fffffff;
      __syncwarp();
    }
    for (int j0 = w.k0; j0 < w.k1; j0 += 16) {
      cp_async_wait<ST - 2>();
      __syncwarp();
      issue(stage == 0 ? ST - 1 : stage - 1);
      if (care < min(j0 + 16, w.k1)) {
        clean_tile<HD, 16, 32>(&sh.kv[stage][1][0], sh.bad, j0, lane);
        __syncwarp();
      }
      rows.take(smem_u32(&sh.kv[stage][0][0]), smem_u32(&sh.kv[stage][1][0]), 0, j0, sl);
      stage = stage == ST - 1 ? 0 : stage + 1;
    }
    rows.finish();
    const int g = lane / 4, t4 = lane % 4;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = w.row0 + g + 8 * r;
      if (i >= w.rows) continue;
      const PaRow x = row_of(a, w, i);
      const long at = x.token * a.hq + x.h;
      const float l = rows.l[r], nat = rows.ref[r] * 0.6931471805599453f;  // natural units outside
      if (careful && l != 0.f) {
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) rows.o[n][2 * r + e] += taken_out<HD>(sh.bad, n * 8 + t4 * 2 + e, rows.seen[r]);
      }
      if (a.direct) {
        // (a row of zeros where nothing counts: o may hold 0 * inf)
        const float f = l > 0.f ? 1.f / l : l;
        bf* out = static_cast<bf*>(a.out) + x.token * a.ldo + static_cast<long>(x.h) * HD + t4 * 2;
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
          *reinterpret_cast<uint32_t*>(out + n * 8) =
              l == 0.f ? 0u : pack_bf16x2(rows.o[n][2 * r] * f, rows.o[n][2 * r + 1] * f);
        if (a.lse && t4 == 0) a.lse[at] = nat + logf(l);
      } else {
        const long slot = static_cast<long>(w.part) * a.b * a.tq * a.hq + at;
        if (t4 == 0) a.part_ml[slot] = make_float2(nat, l);
        if (l != 0.f)
#pragma unroll
          for (int n = 0; n < HD / 8; ++n)
            *reinterpret_cast<float2*>(a.part_o + slot * HD + n * 8 + t4 * 2) =
                make_float2(rows.o[n][2 * r], rows.o[n][2 * r + 1]);
      }
    }
    __syncwarp();  // bad is read before the next piece resets it
  }
  cp_async_wait<0>();
  if (early && blockIdx.x == 0) pdl_wait();
}

template <int HD>
int launch_warp(const PaArgs& a, int prefix_ctas, int own_ctas, bool early, cudaStream_t s) {
  static bool attr = false;
  if (!attr) {
    if (cudaFuncSetAttribute(attn_warp_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(sizeof(WarpShared<HD>))) != cudaSuccess)
      return SB_OPERR_LAUNCH;
    attr = true;
  }
  return launch_pdl(attn_warp_kernel<HD>, dim3(static_cast<unsigned>(prefix_ctas) + own_ctas), dim3(32),
                    sizeof(WarpShared<HD>), s, a, prefix_ctas, early ? 1 : 0) == cudaSuccess
             ? 0
             : SB_OPERR_LAUNCH;
}

template <int HD>
int launch(const PaArgs& a, int prefix_ctas, int own_ctas, bool early, cudaStream_t s) {
  static bool attr = false;
  if (!attr) {
    if (cudaFuncSetAttribute(attn_mma_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(sizeof(MmaShared<HD>))) != cudaSuccess)
      return SB_OPERR_LAUNCH;
    attr = true;
  }
  return launch_pdl(attn_mma_kernel<HD>, dim3(static_cast<unsigned>(prefix_ctas) + own_ctas), dim3(kThreads),
                    sizeof(MmaShared<HD>), s, a, prefix_ctas, early ? 1 : 0) == cudaSuccess
             ? 0
             : SB_OPERR_LAUNCH;
}

}  // namespace

int attn_mma(const PaArgs& a, int hd, int prefix_ctas, int own_ctas, bool early, cudaStream_t s) {
  if (hd == 32) return launch<32>(a, prefix_ctas, own_ctas, early, s);
  if (hd == 64) return launch<64>(a, prefix_ctas, own_ctas, early, s);
  return launch<128>(a, prefix_ctas, own_ctas, early, s);
}

int attn_warp(const PaArgs& a, int hd, int prefix_ctas, int own_ctas, bool early, cudaStream_t s) {
  if (hd == 32) return launch_warp<32>(a, prefix_ctas, own_ctas, early, s);
  if (hd == 64) return launch_warp<64>(a, prefix_ctas, own_ctas, early, s);
  return launch_warp<128>(a, prefix_ctas, own_ctas, early, s);
}

}  // namespace sb
