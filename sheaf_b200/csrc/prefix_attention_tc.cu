// Attention over a paged cache with a shared prefix, many rows a key head
// (bf16), on the tcgen05 tensor cores: with R rows each key brings 2 R
// multiply-adds a byte, so from about 64 rows the products and exponentials
// bound it, not the reading.
//
// A block takes up to 256 rows, two tiles of 128, against tiles of 128 keys;
// 12 warps:
//   warps 0-3, 4-7  softmax of row tile 0, 1: thread = row. S is read from
//             TMEM twice (maximum, then 2^(s - r)); P goes back to TMEM as
//             bf16 over the columns of S it came from, the A operand of P V.
//             The reference r of a row's exponents rises only when a score
//             passes it by 8, so O (in TMEM) is rescaled rarely.
//   warp 8    TMEM owner, one thread issues the UMMAs: for row tile x
//             S_x = Q_x K^T (128 x 128 x HD), O_x += P_x V (128 x HD x 128).
//             While one row tile's softmax runs, the other's products do.
//   warps 9-11  gather Q, K and V rows through the page tables with
//             asynchronous 16-byte copies into 128-byte-swizzled tiles (a
//             page may end anywhere in a tile, which a tiled bulk copy could
//             not follow).
// TMEM: S_0, S_1 (128 columns each), O_0, O_1 (HD each).
#include <algorithm>

#include "prefix_attention.cuh"
#include "sb_kernels.h"
#define SB_PDL_FAMILY 2
#include "sb_launch.cuh"

namespace sb {

namespace {

constexpr int kRows = 128;  // rows of a tile
constexpr int kKeys = 128;  // keys of a tile
constexpr int kSoftWarps = 8, kLoadWarps = 3;  // 12 warps: 168 registers a thread
constexpr int kThreads = 32 * (kSoftWarps + 1 + kLoadWarps);
constexpr int kAtom = 128 * 128;  // bytes of 128 rows x 64 values
constexpr int kLag = 2;           // units of copies in flight behind the newest

template <int HD>
struct Tc {
  static constexpr int kAtoms = HD == 128 ? 2 : 1;
  static constexpr int kTile = kAtoms * kAtom;
  static constexpr int kStages = HD == 128 ? 2 : 3;
  static constexpr int kStageOut = 32 * 64;  // output staging of a warp: 32 rows x 16 floats
  // byte offsets from a 1024-byte boundary
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + 2 * kTile;
  static constexpr int kV = kK + kStages * kTile;
  static constexpr int kOut = kV + kStages * kTile;
  static constexpr int kOffset = kOut + kSoftWarps * kStageOut;  // long [2][kKeys]
  static constexpr int kBad = kOffset + 2 * kKeys * 8;           // int [3 pieces][3][HD]
  static constexpr int kBars = kBad + 9 * HD * 4;
  static constexpr int kNumBars = 2 + 4 * kStages + 6;
  static constexpr int kEnd = kBars + kNumBars * 8 + 32;
  static constexpr int kSmem = kEnd + 1024;
  static constexpr uint32_t kTmemO = 256;  // first column of O_0
};

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void bar_named(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// 16-byte chunk c of row r of a tile (K-major atoms of 64 values).
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return (c >> 3) * kAtom + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// What the values taken out of column c add to a row that sees `seen` keys
// (bad: first key with NaN, +inf, -inf in a column).
template <int HD>
__device__ __forceinline__ float taken_out(const int* bad, int c, int seen) {
  const bool up = bad[HD + c] < seen, down = bad[2 * HD + c] < seen;
  if (bad[c] < seen || (up && down)) return __int_as_float(0x7fffffff);
  return up ? INFINITY : (down ? -INFINITY : 0.f);
}

// The pieces of a block: a run of the prefix's key tiles, or one own piece.
struct Pieces {
  PaRun run;
  int own;
  __device__ __forceinline__ Pieces(const PaArgs& a, int prefix_ctas)
      : run(a.prefix, a.hkv, blockIdx.x), own(static_cast<int>(blockIdx.x) - prefix_ctas) {}
  __device__ __forceinline__ bool next(const PaArgs& a, PaPiece& w) {
    if (own < 0) return run.next(a, blockIdx.x, w);
    if (own == 0x7fffffff) return false;
    w = own_piece(a, own);
    own = 0x7fffffff;
    return true;
  }
};

// `early`: launched beside the kernel before it on the stream, whose own
// predecessors have completed and which writes nothing that this one reads;
// it is waited for at the end.
template <int HD>
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(PaArgs a, int prefix_ctas, int early) {
  extern __shared__ uint8_t smem_raw[];
  using L = Tc<HD>;
  constexpr int ST = L::kStages;
  using bf = __nv_bfloat16;
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::kBars);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* k_full = bars + 2;
  uint64_t* k_empty = k_full + ST;
  uint64_t* v_full = k_empty + ST;
  uint64_t* v_empty = v_full + ST;
  uint64_t* s_full = v_empty + ST;  // [2]
  uint64_t* p_full = s_full + 2;    // [2]
  uint64_t* o_full = p_full + 2;    // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* care = reinterpret_cast<int*>(tmem_slot + 2);  // of the loaders
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    mbar_init(q_full, kLoadWarps);
    mbar_init(q_empty, 1);
    for (int i = 0; i < ST; ++i) {
      mbar_init(&k_full[i], kLoadWarps);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], kLoadWarps);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (!early) pdl_wait();
  if (warp == kSoftWarps) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem = *tmem_slot;
  Pieces pieces(a, prefix_ctas);
  PaPiece w;
  const int tile_rows = static_cast<int>(blockIdx.x) < prefix_ctas ? a.prefix.tile_rows : a.own.tile_rows;

  if (warp > kSoftWarps) {
    // ---- gather ----------------------------------------------------------
    const int tid = threadIdx.x - 32 * (kSoftWarps + 1);
    constexpr int CH = HD / 8, N = kLoadWarps * 32;
    long* offset = reinterpret_cast<long*>(sm + L::kOffset);
    const uint32_t base = smem_u32(sm);
    uint32_t unit = 0, signalled = 0;  // K and V tiles in turn
    int piece = 0, slot = 0;
    uint32_t q_units = 0;  // pieces whose Q is not announced yet
    // The loaders go on after a wait that ran out (the waits then end at once),
    // so that all their warps meet at the same barriers.
    const auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (lane == 0) mbar_wait(bar, parity, a.err, abort_flag);
      __syncwarp();
    };
    const auto signal = [&] {  // the oldest unit has landed for this thread
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        const uint32_t t = signalled >> 1;
        if (!(signalled & 1)) {
          if (q_units) mbar_arrive(q_full);
          mbar_arrive(&k_full[t % ST]);
        } else {
          mbar_arrive(&v_full[t % ST]);
        }
      }
      if (!(signalled & 1)) q_units = 0;
      ++signalled;
    };
    while (pieces.next(a, w)) {
      if (w.k1 <= w.k0) continue;
      const int n = (w.k1 - w.k0 + kKeys - 1) / kKeys;
      // what is in flight is announced before waiting for the last piece's
      // products, which need it
      cp_async_wait<0>();
      while (signalled < unit) signal();
      if (piece > 0) wait(q_empty, (piece - 1) & 1);
      int* bad = reinterpret_cast<int*>(sm + L::kBad) + (piece % 3) * 3 * HD;
      const bool prefix = w.seq < 0;
      const int* table = table_of(a, w);
      const bf* gk = static_cast<const bf*>(a.k) + static_cast<long>(w.head) * a.head_stride;
      const bf* gv = static_cast<const bf*>(a.v) + static_cast<long>(w.head) * a.head_stride;
      for (int i = tid; i < 3 * HD; i += N) bad[i] = 0x7fffffff;
      if (tid == 0) *care = w.k1;
      bar_named(1, N);
      for (int i = tid; i < tile_rows; i += N) {
        if (w.row0 + i >= w.rows) break;
        const int seen = visible(a, prefix, row_of(a, w, w.row0 + i));
        if (seen > w.k0 && seen < w.k1) atomicMin(care, seen);
      }
      // Q: rows past the segment's end are zero
      for (int i = tid; i < tile_rows * CH; i += N) {
        const int r = i / CH, c = i % CH;
        const bool in = w.row0 + r < w.rows;
        long at = 0;
        if (in) {
          const PaRow x = row_of(a, w, w.row0 + r);
          at = x.token * a.ldq + static_cast<long>(x.h) * HD + c * 8;
        }
        cp_async16(base + L::kQ + (r / kRows) * L::kTile + chunk_at(r % kRows, c), static_cast<const bf*>(a.q) + at, in);
      }
      ++q_units;
      const auto locate = [&](int to, int j0) {
        for (int i = tid; i < kKeys; i += N)
          if (j0 + i < w.k1) offset[to * kKeys + i] = key_offset(a, table, j0 + i);
      };
      locate(slot, w.k0);
      bar_named(1, N);
      const int ragged = *care;
      for (int j = 0; j < n; ++j) {
        const int j0 = w.k0 + j * kKeys;
        locate(slot ^ 1, j0 + kKeys);
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // K, then V
          const uint32_t t = unit >> 1, st = t % ST;
          if (t >= ST) wait(half ? &v_empty[st] : &k_empty[st], ((t / ST) & 1) ^ 1);
          const uint32_t tile = base + (half ? L::kV : L::kK) + st * L::kTile;
          const bf* src = half ? gv : gk;
#pragma unroll 8
          for (int i = tid; i < kKeys * CH; i += N) {
            const int r = i / CH, c = i % CH;
            const bool in = j0 + r < w.k1;
            cp_async16(tile + chunk_at(r, c), src + (in ? offset[slot * kKeys + r] + c * 8 : 0), in);
          }
          cp_async_commit();
          if (half && ragged < min(j0 + kKeys, w.k1)) {
            // some row stops inside this tile: values that it must not meet
            // are taken out, each thread its own copies
            cp_async_wait<0>();
            for (int i = tid; i < kKeys * CH; i += N) {
              const int r = i / CH, c = i % CH;
              uint4* p = reinterpret_cast<uint4*>(sm + L::kV + st * L::kTile + chunk_at(r, c));
              const uint4 u = *p;
              uint32_t x[4] = {u.x, u.y, u.z, u.w};
              bool any = false;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t b = (x[e / 2] >> (16 * (e % 2))) & 0xffffu;
                if ((b & 0x7f80u) != 0x7f80u) continue;
                any = true;
                x[e / 2] &= e % 2 ? 0x0000ffffu : 0xffff0000u;
                atomicMin(&bad[((b & 0x7fu) ? 0 : (b >> 15 ? 2 : 1)) * HD + c * 8 + e], j0 + r);
              }
              if (any) *p = make_uint4(x[0], x[1], x[2], x[3]);
            }
          }
          ++unit;
          if (unit - signalled > kLag) {
            cp_async_wait<kLag>();
            signal();
          }
        }
        slot ^= 1;
        bar_named(1, N);  // offsets of the next tile
      }
      ++piece;
    }
    cp_async_wait<0>();
    while (signalled < unit) signal();
  } else if (warp == kSoftWarps) {
    // ---- products --------------------------------------------------------
    if (lane == 0) {
      constexpr uint32_t idS = make_idesc_bf16(128, 128, false, false);
      constexpr uint32_t idO = make_idesc_bf16(128, HD, false, true);
      const uint32_t base = smem_u32(sm);
      uint32_t c = 0;             // key tiles so far
      uint32_t done[2] = {0, 0};  // of each row tile, which a piece may lack
      int piece = 0;
      bool ok = true;
      while (ok && pieces.next(a, w)) {
        if (w.k1 <= w.k0) continue;
        const int n = (w.k1 - w.k0 + kKeys - 1) / kKeys;
        const int tiles = (tile_rows > kRows && w.row0 + kRows < w.rows) ? 2 : 1;
        const auto wait = [&](uint64_t* bar, uint32_t parity) {
          ok = mbar_wait(bar, parity, a.err, abort_flag);
          return ok;
        };
        const auto scores = [&](int x, uint32_t t) {
          const uint32_t q = base + L::kQ + x * L::kTile, k = base + L::kK + (t % ST) * L::kTile;
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t at = (kk >> 2) * kAtom + (kk & 3) * 32;
            umma_f16(tmem + x * 128, make_sw128_desc(q + at, 16, 1024), make_sw128_desc(k + at, 16, 1024), idS, kk > 0);
          }
          umma_commit(&s_full[x]);
        };
        if (!wait(q_full, piece & 1) || !wait(&k_full[c % ST], (c / ST) & 1)) break;
        tc_fence_after();
        for (int x = 0; x < tiles; ++x) scores(x, c);
        umma_commit(&k_empty[c % ST]);
        if (n == 1) umma_commit(q_empty);
        for (int j = 0; j < n && ok; ++j, ++c) {
          const uint32_t st = c % ST;
          if (!wait(&v_full[st], (c / ST) & 1)) break;
          const uint32_t v = base + L::kV + st * L::kTile;
          for (int x = 0; x < tiles; ++x) {
            if (!wait(&p_full[x], done[x] & 1)) break;
            ++done[x];
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < kKeys / 16; ++kk)
              umma_f16_tmem_a(tmem + L::kTmemO + x * HD, tmem + x * 128 + kk * 8,
                              make_sw128_desc(v + kk * 2048, kAtom, 1024), idO, (j > 0 || kk > 0) ? 1u : 0u);
            umma_commit(&o_full[x]);
            if (j + 1 < n) {
              if (x == 0) {
                if (!wait(&k_full[(c + 1) % ST], ((c + 1) / ST) & 1)) break;
                tc_fence_after();
              }
              scores(x, c + 1);
            }
          }
          if (!ok) break;
          umma_commit(&v_empty[st]);
          if (j + 1 < n) {
            umma_commit(&k_empty[(c + 1) % ST]);
            if (j + 2 == n) umma_commit(q_empty);
          }
        }
        ++piece;
      }
      // no commit may arrive on this block's barriers after it has exited
      if (ok && piece > 0) {
        mbar_wait(q_empty, (piece - 1) & 1, a.err, abort_flag);
        for (uint32_t t = c >= ST ? c - ST : 0; t < c; ++t) {
          mbar_wait(&k_empty[t % ST], (t / ST) & 1, a.err, abort_flag);
          mbar_wait(&v_empty[t % ST], (t / ST) & 1, a.err, abort_flag);
        }
      }
    }
    __syncwarp();
  } else {
    // ---- softmax ---------------------------------------------------------
    const int x = warp / 4, quarter = warp % 4;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tS = tmem + lanes + x * 128, tO = tmem + lanes + L::kTmemO + x * HD;
    const float sl = a.scale * 1.4426950408889634f;
    const uint32_t out_tile = smem_u32(sm) + L::kOut + warp * L::kStageOut;
    uint32_t c = 0;
    int piece = 0;
    bool ok = true;
    const auto wait = [&](uint64_t* bar, uint32_t parity) {  // one answer a warp
      ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, a.err, abort_flag));
      tc_fence_after();
      return ok;
    };
    while (ok && pieces.next(a, w)) {
      const bool prefix = w.seq < 0;
      const bool work = w.k1 > w.k0;
      const int n = work ? (w.k1 - w.k0 + kKeys - 1) / kKeys : 0;
      const int i = w.row0 + x * kRows + quarter * 32 + lane;
      const bool mine = x * kRows < tile_rows && i < w.rows;
      int seen = w.k1;
      long at = -1, out_at = 0;  // row among the results, offset of its output
      if (mine) {
        const PaRow r = row_of(a, w, i);
        seen = min(visible(a, prefix, r), w.k1);
        at = r.token * a.hq + r.h;
        out_at = r.token * a.ldo + static_cast<long>(r.h) * HD;
      }
      const int least = __reduce_min_sync(0xffffffffu, seen);
      const bool present = x == 0 || (tile_rows > kRows && w.row0 + kRows < w.rows);
      float ref = -INFINITY, l = 0.f;
      if (present) {
        for (int j = 0; j < n; ++j, ++c) {
          const int j0 = w.k0 + j * kKeys;
          if (!wait(&s_full[x], c & 1)) break;
          const bool part = j0 + kKeys > least;  // some row stops in this tile
          float mx = -INFINITY;
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) {
            uint32_t v[32];
            tmem_ld32(tS + cc * 32, v);
            tmem_wait_ld();
            if (part) {
#pragma unroll
              for (int t = 0; t < 32; ++t)
                if (j0 + cc * 32 + t < seen) mx = fmaxf(mx, __uint_as_float(v[t]));
            } else {
#pragma unroll
              for (int t = 0; t < 32; ++t) mx = fmaxf(mx, __uint_as_float(v[t]));
            }
          }
          mx *= sl;
          if (__any_sync(0xffffffffu, mx > ref + 8.f)) {
            const float to = fmaxf(ref, mx);
            const float f = to == -INFINITY ? 1.f : ex2_approx(ref - to);
            ref = to;
            l *= f;
            if (j > 0) {
              if (!wait(&o_full[x], (c - 1) & 1)) break;
#pragma unroll
              for (int cc = 0; cc < HD / 16; ++cc) {
                uint32_t v[16];
                tmem_ld16(tO + cc * 16, v);
                tmem_wait_ld();
#pragma unroll
                for (int t = 0; t < 16; ++t) v[t] = __float_as_uint(__uint_as_float(v[t]) * f);
                tmem_st16(tO + cc * 16, v);
              }
              tmem_wait_st();
            }
          }
          const float sub = ref == -INFINITY ? 0.f : ref;
          float2 sum = make_float2(0.f, 0.f);
          const float2 sl2 = make_float2(sl, sl), sub2 = make_float2(-sub, -sub);
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) {
            uint32_t v[32], pk[16];
            tmem_ld32(tS + cc * 32, v);
            tmem_wait_ld();
#pragma unroll
            for (int t = 0; t < 32; t += 2) {
              const float2 y =
                  __ffma2_rn(make_float2(__uint_as_float(v[t]), __uint_as_float(v[t + 1])), sl2, sub2);
              float2 p = make_float2(ex2_approx(y.x), ex2_approx(y.y));
              if (part) {
                if (j0 + cc * 32 + t >= seen) p.x = 0.f;
                if (j0 + cc * 32 + t + 1 >= seen) p.y = 0.f;
              }
              sum = __fadd2_rn(sum, p);
              pk[t / 2] = pack_bf16x2(p.x, p.y);
            }
            tmem_st16(tS + cc * 16, pk);
          }
          l += sum.x + sum.y;
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[x]);
        }
        if (!ok) break;
        if (n > 0 && !wait(&o_full[x], (c - 1) & 1)) break;
      }
      const float nat = ref * 0.6931471805599453f;  // natural units outside
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      if (mine) {
        if (a.direct) {
          if (a.lse) a.lse[at] = nat + logf(l);
        } else {
          a.part_ml[static_cast<long>(w.part) * a.b * a.tq * a.hq + at] = make_float2(nat, l);
        }
      }
      // rows leave through shared memory, 64 bytes of 8 rows a store
      const int* bad = reinterpret_cast<const int*>(sm + L::kBad) + (piece % 3) * 3 * HD;
      if (present && (n > 0 || a.direct)) {
        const long row_at = a.direct ? out_at : (static_cast<long>(w.part) * a.b * a.tq * a.hq + at) * HD;
#pragma unroll 1
        for (int cc = 0; cc < HD / 16; ++cc) {
          uint32_t v[16];
          if (n > 0) {
            tmem_ld16(tO + cc * 16, v);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int t = 0; t < 16; ++t) v[t] = 0u;
          }
#pragma unroll
          for (int t = 0; t < 4; ++t)
            st_shared_v4(out_tile + lane * 64 + ((t ^ ((lane >> 1) & 3)) << 4), v[4 * t], v[4 * t + 1], v[4 * t + 2],
                         v[4 * t + 3]);
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r = 8 * k + lane / 4, ch = lane % 4;
            const uint4 u = ld_shared_v4(out_tile + r * 64 + ((ch ^ ((r >> 1) & 3)) << 4));
            const bool theirs = __shfl_sync(0xffffffffu, static_cast<int>(mine), r);
            const float their_l = __shfl_sync(0xffffffffu, l, r);
            const float their_inv = __shfl_sync(0xffffffffu, inv, r);
            const int their_seen = __shfl_sync(0xffffffffu, seen, r);
            const long their_at = __shfl_sync(0xffffffffu, row_at, r);
            if (!theirs) continue;
            float o[4] = {__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w)};
            const int col = cc * 16 + ch * 4;
            if (their_l != 0.f && n > 0) {
#pragma unroll
              for (int e = 0; e < 4; ++e) o[e] += taken_out<HD>(bad, col + e, their_seen);
            }
            if (a.direct) {
              if (their_l == 0.f) o[0] = o[1] = o[2] = o[3] = 0.f;
              *reinterpret_cast<uint2*>(static_cast<bf*>(a.out) + their_at + col) =
                  make_uint2(pack_bf16x2(o[0] * their_inv, o[1] * their_inv),
                             pack_bf16x2(o[2] * their_inv, o[3] * their_inv));
            } else if (their_l != 0.f) {
              *reinterpret_cast<float4*>(a.part_o + their_at + col) = make_float4(o[0], o[1], o[2], o[3]);
            }
          }
          __syncwarp();
        }
      }
      tc_fence_before();  // O is read before the next piece's P is announced
      if (work) ++piece;
    }
  }

  if (early) pdl_wait();
  tc_fence_before();
  __syncthreads();
  if (warp == kSoftWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int HD>
int launch(const PaArgs& a, int prefix_ctas, int own_ctas, bool early, cudaStream_t s) {
  static bool attr = false;
  if (!attr) {
    if (cudaFuncSetAttribute(attn_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tc<HD>::kSmem) !=
        cudaSuccess)
      return SB_OPERR_LAUNCH;
    attr = true;
  }
  // an early launch is one that the launch mask lets overlap; else the stream's order holds
  return launch_pdl(attn_tc_kernel<HD>, dim3(static_cast<unsigned>(prefix_ctas) + own_ctas), dim3(kThreads),
                    Tc<HD>::kSmem, s, a, prefix_ctas, early ? 1 : 0) == cudaSuccess
             ? 0
             : SB_OPERR_LAUNCH;
}

}  // namespace

int attn_tc(const PaArgs& a, int hd, int prefix_ctas, int own_ctas, bool early, cudaStream_t s) {
  if (hd == 32) return launch<32>(a, prefix_ctas, own_ctas, early, s);
  if (hd == 64) return launch<64>(a, prefix_ctas, own_ctas, early, s);
  return launch<128>(a, prefix_ctas, own_ctas, early, s);
}

}  // namespace sb
