// Attention over a paged cache with a shared prefix, few rows a key head
// (bf16): reading the keys bounds it, so the kernel is built around a ring of
// asynchronous copies, and the products run as warp-level m16n8k16 matrix
// instructions on 16 rows, which take a fraction of the copies' time. (The
// tcgen05 kernel's tiles of 128 rows serve larger row blocks.)
//
// A block of 4 warps takes 16, 32 or 64 rows against tiles of 64 keys: with
// 16 rows each warp takes 16 of a tile's keys, with 32 rows two warps share
// the keys of 16 rows, with 64 rows a warp has all keys of its 16. Warps that
// share rows keep their own maxima, sums and outputs and are joined once at
// the end through shared memory.
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

namespace {

constexpr int kKeys = 64;
constexpr int kThreads = 128;

template <int HD>
struct MmaShared {
  static constexpr int kStages = HD == 128 ? 3 : 4;
  static constexpr int kTile = kKeys * HD;  // values
  __nv_bfloat16 kv[kStages][2][kTile];
  long offset[2][kKeys];  // of the keys of the next tiles to load
  int bad[3][HD];         // first key with NaN, +inf, -inf in a column of v
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

// Takes NaN and infinities out of a tile of v (rows j0 .. of the segment) and
// remembers the first key that has one in a column.
template <int HD>
__device__ void clean_tile(MmaShared<HD>& sh, __nv_bfloat16* tile, int j0) {
  for (int i = threadIdx.x; i < MmaShared<HD>::kTile / 8; i += kThreads) {
    const int r = i / (HD / 8), c = i % (HD / 8);
    uint4* p = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(tile) + chunk_at<HD>(r, c));
    uint4 u = *p;
    uint32_t w[4] = {u.x, u.y, u.z, u.w};
    bool any = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t b = (w[e / 2] >> (16 * (e % 2))) & 0xffffu;
      if ((b & 0x7f80u) != 0x7f80u) continue;
      any = true;
      w[e / 2] &= e % 2 ? 0x0000ffffu : 0xffff0000u;
      atomicMin(&sh.bad[(b & 0x7fu) ? 0 : (b >> 15 ? 2 : 1)][c * 8 + e], j0 + r);
    }
    if (any) *p = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// What the values taken out of column c add to a row that sees `seen` keys.
template <int HD>
__device__ __forceinline__ float taken_out(const MmaShared<HD>& sh, int c, int seen) {
  const bool up = sh.bad[1][c] < seen, down = sh.bad[2][c] < seen;
  if (sh.bad[0][c] < seen || (up && down)) return __int_as_float(0x7fffffff);
  return up ? INFINITY : (down ? -INFINITY : 0.f);
}

template <int HD>
__device__ void attend_piece(const PaArgs& a, const PaPiece& w, int tile_rows, MmaShared<HD>& sh) {
  constexpr int KS = HD / 16;  // steps of 16 along head_dim
  constexpr int CH = HD / 8;
  using SH = MmaShared<HD>;
  constexpr int ST = SH::kStages;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int wm = tile_rows / 16;       // warps along the rows
  const int mrow = (warp % wm) * 16;   // this warp's 16 rows of the tile
  const int kgroup = warp / wm;        // its share of a tile's keys: wm groups of 16
  const bool prefix = w.seq < 0;
  const int* table = table_of(a, w);
  using bf = __nv_bfloat16;
  const bf* gk = static_cast<const bf*>(a.k) + static_cast<long>(w.head) * a.head_stride;
  const bf* gv = static_cast<const bf*>(a.v) + static_cast<long>(w.head) * a.head_stride;
  const float sl = a.scale * 1.4426950408889634f;

  // q fragments straight from global memory; rows g and g + 8 of the warp's
  const int g = lane / 4, t4 = lane % 4;
  uint32_t qf[KS][4];
  int seen[2];
  PaRow row[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = w.row0 + mrow + g + 8 * r;
    seen[r] = w.k1;  // a row of no one sees all and is not stored
    if (i < w.rows) {
      row[r] = row_of(a, w, i);
      seen[r] = min(visible(a, prefix, row[r]), w.k1);
      const bf* q = static_cast<const bf*>(a.q) + row[r].token * a.ldq + static_cast<long>(row[r].h) * HD + t4 * 2;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        qf[s][r] = *reinterpret_cast<const uint32_t*>(q + s * 16);
        qf[s][r + 2] = *reinterpret_cast<const uint32_t*>(q + s * 16 + 8);
      }
    } else {
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[s][r] = qf[s][r + 2] = 0u;
    }
  }
  const int warp_lo = __reduce_min_sync(0xffffffffu, min(seen[0], seen[1]));
  // A row that sees some of these keys, but not all, must not meet the values
  // of the others, even as 0 * NaN: tiles past the least such row's count get
  // their values looked through. A row that sees none is dropped by its l = 0.
  const int lo = __reduce_min_sync(
      0xffffffffu, min(seen[0] > w.k0 ? seen[0] : w.k1, seen[1] > w.k0 ? seen[1] : w.k1));

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
  for (int i = tid; i < 3 * HD; i += kThreads) (&sh.bad[0][0])[i] = 0x7fffffff;
  if (tid == 0) sh.care = w.k1;
  locate(0, w.k0);
  __syncthreads();
  if (lane == 0 && lo < w.k1) atomicMin(&sh.care, lo);
  int slot = 0;
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) {
    load(s, slot, w.k0 + s * kKeys);
    locate(slot ^ 1, w.k0 + (s + 1) * kKeys);
    slot ^= 1;
    __syncthreads();
  }

  float o[HD / 8][4];
#pragma unroll
  for (int n = 0; n < HD / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  float ref[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  int stage = 0;
  for (int j0 = w.k0; j0 < w.k1; j0 += kKeys) {
    cp_async_wait<ST - 2>();
    __syncthreads();
    {
      // the slot this tile's predecessor used is free again
      const int ahead = j0 + (ST - 1) * kKeys;
      load(stage == 0 ? ST - 1 : stage - 1, slot, ahead);
      locate(slot ^ 1, ahead + kKeys);
      slot ^= 1;
    }
    const uint32_t sk = smem_u32(&sh.kv[stage][0][0]), sv = smem_u32(&sh.kv[stage][1][0]);
    const int end = min(j0 + kKeys, w.k1);
    if (sh.care < end) {
      clean_tile<HD>(sh, &sh.kv[stage][1][0], j0);
      __syncthreads();
    }
    for (int kg = kgroup * wm; kg < kgroup * wm + wm; ++kg) {
      const int key0 = j0 + kg * 16;
      if (key0 >= end) break;
      float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        // matrices: keys 0-7 and 8-15, each at head_dim 0-7 and 8-15 of the step
        uint32_t kb[4];
        ldmatrix4(kb, sk + chunk_at<HD>(kg * 16 + (lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)));
        mma16816(s[0], qf[ks], kb[0], kb[1]);
        mma16816(s[1], qf[ks], kb[2], kb[3]);
      }
      if (key0 + 16 > warp_lo) {
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
      if (__any_sync(0xffffffffu, mx[0] > ref[0] + 8.f || mx[1] > ref[1] + 8.f)) {
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
      }
      uint32_t pf[4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float sub = ref[r] == -INFINITY ? 0.f : ref[r];
        float p[4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) p[2 * n + e] = ex2_approx(fmaf(s[n][2 * r + e], sl, -sub));
        l[r] += (p[0] + p[1]) + (p[2] + p[3]);
        pf[r] = pack_bf16x2(p[0], p[1]);
        pf[r + 2] = pack_bf16x2(p[2], p[3]);
      }
#pragma unroll
      for (int n = 0; n < KS; ++n) {
        // matrices: keys 0-7 and 8-15 at columns 0-7, then at columns 8-15
        uint32_t vb[4];
        ldmatrix4_t(vb, sv + chunk_at<HD>(kg * 16 + (lane & 15), n * 2 + (lane >> 4)));
        mma16816(o[2 * n], pf, vb[0], vb[1]);
        mma16816(o[2 * n + 1], pf, vb[2], vb[3]);
      }
    }
    stage = stage == ST - 1 ? 0 : stage + 1;
  }
  cp_async_wait<0>();

  // a row's sum over the four lanes that hold its columns of s
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
  }
  __syncthreads();  // the ring is free

  // join the warps that share rows, in the order of their keys
  const int wk = 4 / wm;
  constexpr int P = HD + 4;  // padded row of outputs
  float* buf = reinterpret_cast<float*>(&sh.kv[0][0][0]);  // [kgroup][tile_rows][P]: 64 rows at most
  float2* stat = reinterpret_cast<float2*>(buf + 64 * P);  // [kgroup][tile_rows]
  static_assert(64 * P * 4 + 64 * 8 <= sizeof(sh.kv), "the ring holds the outputs");
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int at = kgroup * tile_rows + mrow + g + 8 * r;
    if (t4 == 0) stat[at] = make_float2(ref[r], l[r]);
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
      *reinterpret_cast<float2*>(&buf[at * P + n * 8 + t4 * 2]) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
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
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < wk; ++k) {
      const float2 st = stat[k * tile_rows + i];
      if (st.y == 0.f) continue;
      const float f = ex2_approx(st.x - m);
      sum = fmaf(st.y, f, sum);
      const float4 u = *reinterpret_cast<const float4*>(&buf[(k * tile_rows + i) * P + c]);
      v.x = fmaf(u.x, f, v.x);
      v.y = fmaf(u.y, f, v.y);
      v.z = fmaf(u.z, f, v.z);
      v.w = fmaf(u.w, f, v.w);
    }
    if (sum != 0.f) {
      const int n = min(visible(a, prefix, x), w.k1);
      v.x += taken_out<HD>(sh, c, n);
      v.y += taken_out<HD>(sh, c + 1, n);
      v.z += taken_out<HD>(sh, c + 2, n);
      v.w += taken_out<HD>(sh, c + 3, n);
    }
    const float nat = m * 0.6931471805599453f;  // natural units outside
    const long at = x.token * a.hq + x.h;
    if (a.direct) {
      const float f = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
      uint2 u;
      u.x = pack_bf16x2(v.x * f, v.y * f);
      u.y = pack_bf16x2(v.z * f, v.w * f);
      *reinterpret_cast<uint2*>(static_cast<bf*>(a.out) + x.token * a.ldo + static_cast<long>(x.h) * HD + c) = u;
      if (a.lse && c == 0) a.lse[at] = nat + logf(sum);
    } else {
      const long slot_at = static_cast<long>(w.part) * a.b * a.tq * a.hq + at;
      if (c == 0) a.part_ml[slot_at] = make_float2(nat, sum);
      if (sum != 0.f) *reinterpret_cast<float4*>(a.part_o + slot_at * HD + c) = v;
    }
  }
}

// Blocks [0, prefix blocks) take runs of the prefix, the others own pieces.
template <int HD>
__global__ void __launch_bounds__(kThreads, HD == 128 ? 2 : 3) attn_mma_kernel(PaArgs a, int prefix_ctas) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  MmaShared<HD>& sh = *reinterpret_cast<MmaShared<HD>*>(smem_raw);
  pdl_wait();
  pdl_trigger();
  const int cta = blockIdx.x;
  if (cta < prefix_ctas) {
    PaRun run(a.prefix, a.hkv, cta);
    PaPiece w;
    while (run.next(a, cta, w)) attend_piece<HD>(a, w, a.prefix.tile_rows, sh);
  } else {
    attend_piece<HD>(a, own_piece(a, cta - prefix_ctas), a.own.tile_rows, sh);
  }
}

template <int HD>
int launch(const PaArgs& a, int prefix_ctas, int own_ctas, cudaStream_t s) {
  static bool attr = false;
  if (!attr) {
    if (cudaFuncSetAttribute(attn_mma_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(sizeof(MmaShared<HD>))) != cudaSuccess)
      return SB_OPERR_LAUNCH;
    attr = true;
  }
  return launch_pdl(attn_mma_kernel<HD>, dim3(static_cast<unsigned>(prefix_ctas) + own_ctas), dim3(kThreads),
                    sizeof(MmaShared<HD>), s, a, prefix_ctas) == cudaSuccess
             ? 0
             : SB_OPERR_LAUNCH;
}

}  // namespace

int attn_mma(const PaArgs& a, int hd, int prefix_ctas, int own_ctas, cudaStream_t s) {
  if (hd == 32) return launch<32>(a, prefix_ctas, own_ctas, s);
  if (hd == 64) return launch<64>(a, prefix_ctas, own_ctas, s);
  return launch<128>(a, prefix_ctas, own_ctas, s);
}

}  // namespace sb
