// Attention over a paged cache with a shared prefix, many rows a key head
// (bf16), on the tcgen05 tensor cores: with R rows each key brings 2 R
// multiply-adds a byte, so from about 64 rows the products and exponentials
// bound it, not the reading.
//
// What bounds it: per key tile and SM, 32 UMMAs of 64 cycles against 32768
// exponentials at 16 a cycle, 2050 cycles each; measured 3690, because a row
// tile's softmax (1620) and its products with their commits and waits (2070)
// follow one another, with the other row tile half a period behind. 512 x 32
// queries behind 16384 keys, 137 GFLOP: 134 us, 0.63 of the measured bf16 peak,
// with the join (under the power cap, at 1745 MHz, 151).
// (7 of 16 exponentials as polynomials in FMAs: 4140 cycles.)
//
// A block takes up to 256 rows, two tiles of 128, against tiles of 128 keys;
// 12 warps:
//   warps 0-3, 4-7  softmax of row tile 0, 1: thread = row; P goes back to TMEM as bf16 over the
//             columns of S it came from, the A operand of P V. (One bf16, with an
//             error of the outputs against 64 bits of 2.3e-3 where the sum of two
//             gives the outputs' own rounding, 1.7e-3: a second term would double
//             the products with V in a kernel that products bound. From 17 rows on
//             this holds where reading bounds it, too.) The reference
//             r of a row's exponents 2^(s - r) rises only when their sum over a
//             tile passes 2^15, so O (in TMEM) is rescaled rarely.
//   warp 8    TMEM owner, one thread issues the UMMAs: for row tile x
//             S_x = Q_x K^T (128 x 128 x HD), O_x += P_x V (128 x HD x 128).
//             While one row tile's softmax runs, the other's products do.
//   warps 9, 10  copy K, V through the page tables: a tiled bulk copy for each
//             run of rows that lies in one page whatever the tile's place (the
//             largest power of two that divides the page), a lane each. (With
//             one warp for both, K waited behind V for room: 512 queries of 32
//             heads behind 16384 keys took 271 us, with two 210. 16-byte
//             asynchronous copies by 96 threads before that: 446.)
//   warp 11   looks through the tiles of V in which a row stops (below).
// The softmax warps gather their rows of Q, those of the next piece while the
// last products of this one run.
// With at most 128 rows and several key tiles a block, the two softmax groups
// take the same rows and the key tiles in turn, each with an output of its own
// (two parts).
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
constexpr int kSoftWarps = 8;
constexpr int kThreads = 32 * (kSoftWarps + 4);  // 168 registers a thread
// Registers a thread: a softmax thread holds its row's 128 scores. Together
// what the launch gave: 256 x 208 + 128 x 88 = 384 x 168.
constexpr int kSoftRegs = 208, kOtherRegs = 88;
constexpr int kAtom = 128 * 128;  // bytes of 128 rows x 64 values

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
  static constexpr int kBad = kOut + kSoftWarps * kStageOut;  // int [2][3][HD]
  static constexpr int kFound = kBad + 2 * 3 * HD * 4;  // int: the piece that kBad is about, plus one
  static constexpr int kDone = kFound + 16;         // int [softmax warps]: pieces finished
  static constexpr int kBars = kDone + 4 * kSoftWarps;
  static constexpr int kNumBars = 2 + 5 * kStages + 6;
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
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
// 16-byte chunk c of row r of a tile (K-major atoms of 64 values).
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return (c >> 3) * kAtom + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// What the values taken out of column c add to a row that sees `seen` keys
// (bad: first key with NaN, +inf, -inf in a column; where key tiles are dealt
// out to the two softmax groups, among a group's own ones: a value counts in
// the part of its tile, and nothing is added while a group reads).
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
      : run(a.prefix, a.hkv.d, blockIdx.x), own(static_cast<int>(blockIdx.x) - prefix_ctas) {}
  __device__ __forceinline__ bool next(const PaArgs& a, PaPiece& w) {
    if (own < 0) return run.next(a, blockIdx.x, w);
    if (own == 0x7fffffff) return false;
    w = own_piece(a, own);
    own = 0x7fffffff;
    return true;
  }
};

// From this key on some row of the piece stops before the piece does. Such a
// row must not meet the values behind its last key, even as 0 * NaN, so the
// tiles of V from there on get their NaN and infinities taken out, to be added
// to the rows that see them at the end. (A row that sees no key of the piece
// is dropped by its l = 0.) All lanes of a warp get the answer.
__device__ __forceinline__ int care_of(const PaArgs& a, const PaPiece& w, int tile_rows) {
  const int rows = min(tile_rows, w.rows - w.row0);
  if (w.seq >= 0) {  // successive queries of one sequence: each sees one key more, or as many
    const int seen = visible(a, false, row_of(a, w, w.row0));
    return min(max(seen, w.k0 + 1), w.k1);
  }
  int care = w.k1;
#pragma unroll
  for (int n = 0; n < 8; ++n) {  // 256 rows; the loads are in flight together
    const int i = min(n * 32 + static_cast<int>(threadIdx.x % 32), rows - 1);
    const int seen = visible(a, true, row_of(a, w, w.row0 + i));
    if (seen > w.k0) care = min(care, seen);
  }
  return __reduce_min_sync(0xffffffffu, care);
}
// Whether the values of tile j0 are looked through: a row stops inside it, or
// the piece does (what lies behind is then whatever shared memory holds).
__device__ __forceinline__ bool special(const PaPiece& w, int care, int j0) {
  return care < j0 + kKeys;
}

// `early`: see attn_tc's declaration.
template <int HD>
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(const __grid_constant__ CUtensorMap tm_k,
                                                              const __grid_constant__ CUtensorMap tm_v, PaArgs a,
                                                              int prefix_ctas, int early) {
  extern __shared__ uint8_t smem_raw[];
  using L = Tc<HD>;
  constexpr int ST = L::kStages;
  using bf = __nv_bfloat16;
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::kBars);
  uint64_t* q_full = bars;  // [2]
  uint64_t* k_full = bars + 2;
  uint64_t* k_empty = k_full + ST;
  uint64_t* v_full = k_empty + ST;
  uint64_t* v_empty = v_full + ST;
  uint64_t* v_raw = v_empty + ST;   // a special tile of V has landed
  uint64_t* s_full = v_raw + ST;    // [2]
  uint64_t* p_full = s_full + 2;    // [2]
  uint64_t* o_full = p_full + 2;    // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&v_raw[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    *abort_flag = 0;
    *reinterpret_cast<int*>(sm + L::kFound) = 0;
    for (int i = 0; i < kSoftWarps; ++i) reinterpret_cast<int*>(sm + L::kDone)[i] = 0;
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
  const bool of_prefix = static_cast<int>(blockIdx.x) < prefix_ctas;
  const int tile_rows = of_prefix ? a.prefix.tile_rows : a.own.tile_rows;
  // one row tile, whose key tiles go to the two softmax groups in turn
  const bool deal = (of_prefix ? a.prefix.slots : a.own.slots) == 2;

  if (warp >= kSoftWarps) regs_down<kOtherRegs>();
  if (warp == kSoftWarps + 1 || warp == kSoftWarps + 2) {
    // ---- copies of K, V ----------------------------------------------------
    const bool values = warp == kSoftWarps + 2;
    const CUtensorMap* map = values ? &tm_v : &tm_k;
    uint64_t* full = values ? v_full : k_full;
    uint64_t* empty = values ? v_empty : k_empty;
    const int boxes = kKeys / a.box_rows;  // of 64 values' width
    const int row = lane % boxes * a.box_rows, atom = lane / boxes;  // this lane's box of a tile
    const bool active = atom < L::kAtoms;
    const uint32_t bytes = a.box_rows * 128;
    const uint32_t to = smem_u32(sm) + (values ? L::kV : L::kK) + atom * kAtom + row * 128;
    uint32_t t = 0;  // tiles so far
    bool ok = true;
    while (ok && pieces.next(a, w)) {
      if (w.k1 <= w.k0) continue;
      const int* table = table_of(a, w);
      int page = active && w.k0 + row < w.k1 ? page_of(a, table, w.k0 + row) : 0;
      const int care = values ? care_of(a, w, tile_rows) : 0;
      for (int j0 = w.k0; j0 < w.k1; j0 += kKeys, ++t) {
        const bool mine = active && j0 + row < w.k1;
        const int in_page = j0 + row - static_cast<int>(a.page_rows(j0 + row) * a.page_rows.d);
        const uint32_t all = __popc(__ballot_sync(0xffffffffu, mine)) * bytes;
        const int this_page = page;
        if (active && j0 + kKeys + row < w.k1) page = page_of(a, table, j0 + kKeys + row);
        const uint32_t st = t % ST;
        if (t >= ST) {
          ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], ((t / ST) & 1) ^ 1, a.err, abort_flag));
          if (!ok) break;
        }
        uint64_t* bar = values && special(w, care, j0) ? &v_raw[st] : &full[st];
        if (lane == 0) mbar_arrive_expect_tx(bar, all);
        __syncwarp();
        if (mine) tma_load_4d(to + st * L::kTile, map, bar, atom * 64, w.head, in_page, this_page);
      }
    }
    if (!ok) {  // copies in flight land before the block may end, or a second passes
      __syncwarp();
      const unsigned long long t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 1000000000ull) {
      }
    }
  } else if (warp > kSoftWarps + 2) {
    // ---- special tiles of V ------------------------------------------------
    constexpr int CH = HD / 8;
    uint32_t t = 0, raw[ST] = {};  // tiles so far, special ones of a stage
    int piece = 0;
    bool ok = true;
    while (ok && pieces.next(a, w)) {
      if (w.k1 <= w.k0) continue;
      const int care = care_of(a, w, tile_rows);
      for (int j0 = w.k0; j0 < w.k1; j0 += kKeys, ++t) {
        if (!special(w, care, j0)) continue;
        const uint32_t st = t % ST;
#pragma unroll
        for (int s = 0; s < ST; ++s)
          if (static_cast<uint32_t>(s) == st) ok = mbar_wait(&v_raw[st], raw[s]++ & 1, a.err, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        uint8_t* tile = sm + L::kV + st * L::kTile;
        const int rows = min(kKeys, w.k1 - j0);
        // rows behind the piece's end, which nothing was copied to, are zero
        for (int i = rows * CH + lane; i < kKeys * CH; i += 32)
          *reinterpret_cast<uint4*>(tile + chunk_at(i / CH, i % CH)) = make_uint4(0u, 0u, 0u, 0u);
        if (care < j0 + rows) {
          // an exponent of all ones carries into the bit above
          const auto odd = [](uint32_t x) { return (x & 0x7f807f80u) + 0x00800080u; };
          uint32_t carry = 0;
#pragma unroll 8
          for (int i = lane; i < rows * CH; i += 32) {
            const uint4 u = *reinterpret_cast<const uint4*>(tile + chunk_at(i / CH, i % CH));
            carry |= odd(u.x) | odd(u.y) | odd(u.z) | odd(u.w);
          }
          const bool any = (carry & 0x80008000u) != 0;
          if (__any_sync(0xffffffffu, any)) {
            int* bad = reinterpret_cast<int*>(sm + L::kBad);
            volatile int* found = reinterpret_cast<volatile int*>(sm + L::kFound);
            volatile int* finished = reinterpret_cast<volatile int*>(sm + L::kDone);
            if (*found != piece + 1) {  // the first of the piece: the pieces before are read to the end
              const unsigned long long t0 = global_timer_ns();
              while (!__all_sync(0xffffffffu, lane >= kSoftWarps || finished[lane] >= piece)) {
                if (global_timer_ns() - t0 > kWaitLimitNs) {
                  if (a.err) atomicExch(a.err, kErrBarrierTimeout);
                  *abort_flag = 1;
                  break;
                }
              }
              for (int i = lane; i < 2 * 3 * HD; i += 32) bad[i] = 0x7fffffff;
              __syncwarp();
              if (lane == 0) *found = piece + 1;
              __syncwarp();
            }
            if (deal) bad += ((j0 - w.k0) / kKeys & 1) * 3 * HD;
            for (int i = lane; i < rows * CH; i += 32) {
              const int r = i / CH, c = i % CH;
              uint4* p = reinterpret_cast<uint4*>(tile + chunk_at(r, c));
              const uint4 u = *p;
              uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t b = (x[e / 2] >> (16 * (e % 2))) & 0xffffu;
                if ((b & 0x7f80u) != 0x7f80u) continue;
                x[e / 2] &= e % 2 ? 0x0000ffffu : 0xffff0000u;
                atomicMin(&bad[((b & 0x7fu) ? 0 : (b >> 15 ? 2 : 1)) * HD + c * 8 + e], j0 + r);
              }
              *p = make_uint4(x[0], x[1], x[2], x[3]);
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[st]);
      }
      ++piece;
    }
  } else if (warp == kSoftWarps) {
    // ---- products --------------------------------------------------------
    // The whole warp runs this with the same values and one lane issues, so
    // that the descriptors live in uniform registers; a step's descriptor is
    // the tile's plus a constant.
    constexpr uint32_t idS = make_idesc_bf16(128, 128, false, false);
    constexpr uint32_t idO = make_idesc_bf16(128, HD, false, true);
    constexpr uint32_t kStep = L::kTile >> 4;
    const uint32_t base = smem_u32(sm);
    const uint64_t dq = make_sw128_desc(base + L::kQ, 16, 1024), dk = make_sw128_desc(base + L::kK, 16, 1024);
    const uint64_t dv = make_sw128_desc(base + L::kV, kAtom, 1024);
    const bool one = elect_one_lane();
    uint32_t c = 0, kst = 0, kph = 0, vst = 0, vph = 0;  // key tiles so far; stages and their phases
    uint32_t done[2] = {0, 0};   // key tiles of each row tile, which a piece may lack
    uint32_t begun[2] = {0, 0};  // pieces
    bool ok = true;
    const auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, a.err, abort_flag));
      tc_fence_after();
      return ok;
    };
    const auto scores = [&](int x) {
      if (one) {
        const uint64_t q = dq + x * kStep, k = dk + kst * kStep;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t at = ((kk >> 2) * kAtom + (kk & 3) * 32) >> 4;
          umma_f16(tmem + x * 128, q + at, k + at, idS, kk > 0);
        }
        umma_commit(&s_full[x]);
      }
    };
    const auto product = [&](int x, bool more) {  // O_x (+)= P_x V
      if (one) {
        const uint64_t v = dv + vst * kStep;
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          umma_f16_tmem_a(tmem + L::kTmemO + x * HD, tmem + x * 128 + kk * 8, v + ((kk * 2048) >> 4), idO,
                          (more || kk > 0) ? 1u : 0u);
        umma_commit(&o_full[x]);
      }
    };
    const auto next_k = [&] {  // the products issued are the last to read this stage
      if (one) umma_commit(&k_empty[kst]);
      kst = kst + 1 == ST ? 0 : kst + 1;
      kph ^= kst == 0;
    };
    const auto next_v = [&] {
      if (one) umma_commit(&v_empty[vst]);
      vst = vst + 1 == ST ? 0 : vst + 1;
      vph ^= vst == 0;
    };
    while (ok && pieces.next(a, w)) {
      if (w.k1 <= w.k0) continue;
      const int n = (w.k1 - w.k0 + kKeys - 1) / kKeys;
      if (deal) {
        // key tile j for softmax group j % 2
        for (int j = 0; j < min(n, 2); ++j) {
          if (!wait(&k_full[kst], kph) || !wait(&q_full[j], begun[j]++ & 1)) break;
          scores(j);
          next_k();
        }
        if (!ok) break;
        for (int j = 0; j < n; ++j, ++c) {
          const int x = j & 1;
          if (!wait(&v_full[vst], vph) || !wait(&p_full[x], done[x]++ & 1)) break;
          product(x, j > 1);
          next_v();
          if (j + 2 < n) {
            if (!wait(&k_full[kst], kph)) break;
            scores(x);
            next_k();
          }
        }
        continue;
      }
      const int tiles = tile_rows > kRows && w.row0 + kRows < w.rows ? 2 : 1;
      if (!wait(&k_full[kst], kph)) break;
      for (int x = 0; x < tiles; ++x) {
        if (!wait(&q_full[x], begun[x]++ & 1)) break;
        scores(x);
      }
      if (!ok) break;
      for (int j = 0; j < n; ++j, ++c) {
        next_k();
        if (!wait(&v_full[vst], vph)) break;
        for (int x = 0; x < tiles; ++x) {
          if (!wait(&p_full[x], done[x]++ & 1)) break;
          product(x, j > 0);
          if (j + 1 < n) {
            if (x == 0 && !wait(&k_full[kst], kph)) break;
            scores(x);
          }
        }
        if (!ok) break;
        next_v();
      }
    }
    // no commit may arrive on this block's barriers after it has exited
    if (ok)
      for (uint32_t t = c >= ST ? c - ST : 0; t < c; ++t)
        if (!wait(&k_empty[t % ST], (t / ST) & 1) || !wait(&v_empty[t % ST], (t / ST) & 1)) break;
  } else {
    // ---- softmax ---------------------------------------------------------
    regs_up<kSoftRegs>();
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
    // this thread's row of a piece
    struct Mine {
      bool in;           // has a row
      bool none;         // the row sees none of the piece's keys
      int tiles;         // key tiles that this group takes
      int seen;
      long at, out_at;   // among the results; offset of its output
    };
    const auto row_in = [&](const PaPiece& p) {
      Mine m;
      const int i = p.row0 + (deal ? 0 : x * kRows) + quarter * 32 + lane;
      m.in = i < p.rows && (deal || x == 0 || tile_rows > kRows);
      m.tiles = (max(p.k1 - p.k0, 0) + kKeys - 1) / kKeys;
      if (deal)
        m.tiles = (m.tiles + 1 - x) / 2;
      else if (x == 1 && (tile_rows == kRows || p.row0 + kRows >= p.rows))
        m.tiles = 0;
      m.none = false;
      m.seen = p.k1;  // a row that sees nothing is let go along, and dropped at the end
      m.at = 0;
      m.out_at = 0;
      long q_at = -1;
      PaRow r;
      if (m.in) {
        r = row_of(a, p, i);
        m.at = r.token * a.hq + r.h;
        m.out_at = r.token * a.ldo + static_cast<long>(r.h) * HD;
        q_at = r.token * a.ldq + static_cast<long>(r.h) * HD;
      }
      // this warp's rows of Q; rows past the segment's end are zero. The
      // row tile's last scores are done: Q is free.
      if (m.tiles > 0) {
        constexpr int CH = HD / 8, RPI = 32 / CH;  // rows an instruction
#pragma unroll
        for (int n = 0; n < 32 / RPI; ++n) {
          const int r = n * RPI + lane / CH, ch = lane % CH;
          const long from = __shfl_sync(0xffffffffu, q_at, r);
          cp_async16(smem_u32(sm) + L::kQ + x * L::kTile + chunk_at(quarter * 32 + r, ch),
                     static_cast<const bf*>(a.q) + (from < 0 ? 0 : from + ch * 8), from >= 0);
        }
      }
      cp_async_commit();
      if (m.in) {
        const int seen = visible(a, p.seq < 0, r);
        m.none = seen <= p.k0;
        if (!m.none) m.seen = min(seen, p.k1);
      }
      return m;
    };
    const auto announce_q = [&](const Mine& m) {
      cp_async_wait<0>();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && m.tiles > 0) mbar_arrive(&q_full[x]);
    };
    PaPiece next_w;
    bool more = pieces.next(a, next_w);
    Mine next_mine = {};
    if (more) {
      next_mine = row_in(next_w);
      announce_q(next_mine);
    }
    while (ok && more) {
      w = next_w;
      const Mine mine = next_mine;
      const int seen = mine.seen;
      const int least = __reduce_min_sync(0xffffffffu, seen);
      float ref = -INFINITY, l = 0.f;
      bool open = true;  // some row has no reference yet: every score it has seen is -inf
      bool far = false;  // some row's reference is far out
      for (int j = 0; j < mine.tiles; ++j, ++c) {
        const int j0 = w.k0 + (deal ? 2 * j + x : j) * kKeys;
        if (!wait(&s_full[x], c & 1)) break;
        const bool part = j0 + kKeys > least;  // some row stops in this tile
        // Scores go to p = 2^(s - ref) without their maximum being looked
        // for. Only until every row has a reference (next loop; mostly at a
        // piece's first tile) and where a row's sum passes 2^15 is it raised;
        // in the latter case O is rescaled and p taken again from the scores,
        // still in registers.
        if (open || part) {
          // keys that a row does not see get their scores out of the way
          float mx = -INFINITY;
#pragma unroll 1
          for (int cc = 0; cc < 8; ++cc) {
            uint32_t u[16];
            tmem_ld16(tS + cc * 16, u);
            tmem_wait_ld();
            const int limit = seen - j0 - cc * 16;
#pragma unroll
            for (int t = 0; t < 16; ++t) {
              if (t >= limit) u[t] = __float_as_uint(-INFINITY);
              mx = fmaxf(mx, __uint_as_float(u[t]));
            }
            if (part) tmem_st16(tS + cc * 16, u);
          }
          if (part) tmem_wait_st();
          if (open) {
            if (ref == -INFINITY) ref = mx * sl;
            open = __any_sync(0xffffffffu, ref == -INFINITY && j0 + kKeys < seen);
            far = __any_sync(0xffffffffu, far_out(ref));
          }
        }
        float by = sl;
        if (__builtin_expect(far, 0)) {
#pragma unroll 1
          for (int cc = 0; cc < 8; ++cc) {
            uint32_t u[16];
            tmem_ld16(tS + cc * 16, u);
            tmem_wait_ld();
#pragma unroll
            for (int t = 0; t < 16; ++t) u[t] = __float_as_uint(__uint_as_float(u[t]) * sl);
            tmem_st16(tS + cc * 16, u);
          }
          tmem_wait_st();
          by = 1.f;
        }
        uint32_t v[4][32];
        float2 sum[2];
        const auto exps = [&](int cc, float by) {
          const float2 by2 = make_float2(by, by);
          const float sub = ref == -INFINITY ? 0.f : ref;
          const float2 sub2 = make_float2(-sub, -sub);
          uint32_t pk[16];
#pragma unroll
          for (int t = 0; t < 16; ++t) {
            const float2 y = __ffma2_rn(
                make_float2(__uint_as_float(v[cc][2 * t]), __uint_as_float(v[cc][2 * t + 1])), by2, sub2);
            const float2 p = make_float2(ex2_approx(y.x), ex2_approx(y.y));
            sum[t & 1] = __fadd2_rn(sum[t & 1], p);
            pk[t] = pack_bf16x2(p.x, p.y);
          }
          tmem_st16(tS + cc * 16, pk);  // over scores that have been read
        };
        const auto total = [&] { return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y); };
        // 32 scores at a time, the next on their way meanwhile
        sum[0] = sum[1] = make_float2(0.f, 0.f);
        tmem_ld32(tS, v[0]);
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          tmem_wait_ld();
          if (cc < 3) tmem_ld32(tS + (cc + 1) * 32, v[cc + 1]);
          exps(cc, by);
        }
        float tile_l = total();
        // A NaN is left as it is.
        if (__builtin_expect(__any_sync(0xffffffffu, tile_l > 32768.f), 0)) {
          float m[2] = {ref, -INFINITY};
#pragma unroll
          for (int cc = 0; cc < 4; ++cc)
#pragma unroll
            for (int t = 0; t < 32; t += 2) {
              const float s0 = __uint_as_float(v[cc][t]) * by, s1 = __uint_as_float(v[cc][t + 1]) * by;
              m[0] = fmaxf(m[0], s0);
              m[1] = fmaxf(m[1], s1);
              v[cc][t] = __float_as_uint(s0);
              v[cc][t + 1] = __float_as_uint(s1);
            }
          const float mx = fmaxf(m[0], m[1]);
          const float f = mx == -INFINITY ? 1.f : ex2_approx(ref - mx);
          ref = mx;
          far = __any_sync(0xffffffffu, far_out(ref));
          l *= f;
          if (j > 0) {
            if (!wait(&o_full[x], (c - 1) & 1)) break;
#pragma unroll 1
            for (int cc = 0; cc < HD / 16; ++cc) {
              uint32_t u[16];
              tmem_ld16(tO + cc * 16, u);
              tmem_wait_ld();
#pragma unroll
              for (int t = 0; t < 16; ++t) u[t] = __float_as_uint(__uint_as_float(u[t]) * f);
              tmem_st16(tO + cc * 16, u);
            }
          }
          sum[0] = sum[1] = make_float2(0.f, 0.f);
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) exps(cc, 1.f);
          tile_l = total();
        }
        l += tile_l;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[x]);
      }
      if (!ok) break;
      if (mine.none) {
        ref = -INFINITY;
        l = 0.f;
      }
      more = pieces.next(a, next_w);
      if (more) next_mine = row_in(next_w);
      if (mine.tiles > 0 && !wait(&o_full[x], (c - 1) & 1)) break;
      const float nat = ref * 0.6931471805599453f;  // natural units outside
      const long part_at = static_cast<long>(w.part + (deal ? x : 0)) * a.b * a.tq * a.hq + mine.at;
      if (mine.in) {
        if (a.direct) {
          if (a.lse) a.lse[mine.at] = nat + logf(l);
        } else {
          a.part_ml[part_at] = make_float2(nat, l);
        }
      }
      // rows leave through shared memory, 64 bytes of 8 rows a store
      if (mine.tiles > 0 || a.direct) {
        const bool some = mine.tiles > 0 && *reinterpret_cast<volatile const int*>(sm + L::kFound) == piece + 1;
        const int* bad = reinterpret_cast<const int*>(sm + L::kBad) + (deal ? x * 3 * HD : 0);
        const long row_at = !mine.in || (!a.direct && l == 0.f) ? -1 : (a.direct ? mine.out_at : part_at * HD);
        const float scale = a.direct ? (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) : 1.f;
        long their_at[4];
        float their_scale[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          their_at[k] = __shfl_sync(0xffffffffu, row_at, 8 * k + lane / 4);
          their_scale[k] = __shfl_sync(0xffffffffu, scale, 8 * k + lane / 4);
        }
        uint32_t ahead[16];
        tmem_ld16(tO, ahead);
#pragma unroll 1
        for (int cc = 0; cc < HD / 16; ++cc) {
          uint32_t v[16];
          tmem_wait_ld();
#pragma unroll
          for (int t = 0; t < 16; ++t) v[t] = ahead[t];
          if (cc + 1 < HD / 16) tmem_ld16(tO + (cc + 1) * 16, ahead);
          if (some && l != 0.f) {
#pragma unroll
            for (int t = 0; t < 16; ++t)
              v[t] = __float_as_uint(__uint_as_float(v[t]) + taken_out<HD>(bad, cc * 16 + t, seen));
          }
#pragma unroll
          for (int t = 0; t < 4; ++t)
            st_shared_v4(out_tile + lane * 64 + ((t ^ ((lane >> 1) & 3)) << 4), v[4 * t], v[4 * t + 1], v[4 * t + 2],
                         v[4 * t + 3]);
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r = 8 * k + lane / 4, ch = lane % 4, col = cc * 16 + ch * 4;
            const uint4 u = ld_shared_v4(out_tile + r * 64 + ((ch ^ ((r >> 1) & 3)) << 4));
            if (their_at[k] < 0) continue;
            if (a.direct) {
              const float f = their_scale[k];
              uint2 o = make_uint2(pack_bf16x2(__uint_as_float(u.x) * f, __uint_as_float(u.y) * f),
                                   pack_bf16x2(__uint_as_float(u.z) * f, __uint_as_float(u.w) * f));
              if (f == 0.f) o = make_uint2(0u, 0u);  // a row that saw nothing
              *reinterpret_cast<uint2*>(static_cast<bf*>(a.out) + their_at[k] + col) = o;
            } else {
              *reinterpret_cast<uint4*>(a.part_o + their_at[k] + col) = u;
            }
          }
          __syncwarp();
        }
      }
      tc_fence_before();  // O is read before the next piece's P is announced
      if (more) announce_q(next_mine);
      if (w.k1 > w.k0) {
        ++piece;
        __syncwarp();
        if (lane == 0) reinterpret_cast<volatile int*>(sm + L::kDone)[warp] = piece;
      }
    }
    cp_async_wait<0>();
  }

  if (early && blockIdx.x == 0) pdl_wait();
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
  alignas(64) CUtensorMap tk, tv;
  if (!cache_map(&tk, a.k, a, HD) || !cache_map(&tv, a.v, a, HD)) return SB_OPERR_TMA;
  return launch_pdl(attn_tc_kernel<HD>, dim3(static_cast<unsigned>(prefix_ctas) + own_ctas), dim3(kThreads),
                    Tc<HD>::kSmem, s, tk, tv, a, prefix_ctas, early ? 1 : 0) == cudaSuccess
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
