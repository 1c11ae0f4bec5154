// Log probabilities of given tokens, the entropy of their distributions, the
// most likely alternatives, and the VJP.
//
// With z = x / temperature, a row of v logits, t its given token:
//   lse = log sum_j exp z_j      logp = z_t - lse
//   H   = - sum_j p_j log p_j    p = exp(z - lse)
// One pass keeps, per thread, an integer reference R >= the largest y of what
// it has seen, y = z log2(e), and S = sum 2^(y - R), W = sum 2^(y - R) (y - R):
//   lse = ln2 (R + log2 S),   H = ln2 (log2 S - W / S)
// y - R is one fused multiply-add with a single rounding, and references differ
// by whole numbers, so joining two threads' sums scales by exact powers of two.
// Logits below -1e29 count as -inf there. A row with nothing else, or whose
// reference passes 2^22, where floats thin out to whole numbers and S could end
// up far below 1, is taken again by differences of the logits themselves.
//
// The k best (larger value first, then lower index) come from the same pass:
// each thread remembers its largest 16-byte vector. The k-th largest of 64
// groups of threads (32 single ones, where a warp has the row) bounds the k-th
// best logit from below, so only what the few threads saw whose own best
// reaches that bound is looked at again (from L2, by all threads), and only
// logits that reach it become candidates: about 64 ln(64 / (64 - k)) of them.
//
// Reading the logits bounds it: 8192 x 50304 bf16, 824 MB, take 126 us at the
// measured copy rate, and 164-170 us without alternatives, 185 with 8 where calls
// follow one another, 195 (0.64) each with new logits. What is left: the
// exponentials alone take 0.57 of the time on their unit, and a block does not
// read while it joins a row's statistics and looks up the alternatives. The VJP
// reads and writes once: 4096 x 50304 in 147 us (0.86) and 152 likewise.
#include <cuda_bf16.h>

#include <algorithm>
#include <cfloat>

#include "sb_cache.h"
#include "sb_kernels.h"
#include "sb_ptx.cuh"
#define SB_PDL_FAMILY 1
#include "sb_launch.cuh"

namespace sb {

int num_sms_cached();

namespace {

using u64 = unsigned long long;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -INFINITY;

__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int N = 4;  // values of a 16-byte vector
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x);
    f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z);
    f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  // The largest value, or NaN.
  static __device__ __forceinline__ float most(const uint4& u) {
    return max_nan(max_nan(__uint_as_float(u.x), __uint_as_float(u.y)),
                   max_nan(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  // Values below -1e30 become that; NaN stays.
  static __device__ __forceinline__ uint4 floored(uint4 u) {
    const auto f = [](uint32_t x) { return __float_as_uint(max_nan(__uint_as_float(x), -1e30f)); };
    return make_uint4(f(u.x), f(u.y), f(u.z), f(u.w));
  }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ __nv_bfloat162 two(uint32_t x) { return *reinterpret_cast<__nv_bfloat162*>(&x); }
  static __device__ __forceinline__ float most(const uint4& u) {
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(two(u.x), two(u.y)), __hmax2_nan(two(u.z), two(u.w)));
    return max_nan(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ uint4 floored(uint4 u) {
    const __nv_bfloat162 lowest = __float2bfloat162_rn(-1e30f);
    const auto f = [&](uint32_t x) {
      const __nv_bfloat162 m = __hmax2_nan(two(x), lowest);
      return *reinterpret_cast<const uint32_t*>(&m);
    };
    return make_uint4(f(u.x), f(u.y), f(u.z), f(u.w));
  }
};

constexpr uint32_t kNanImage = 0xfffffff0u;  // above that of +inf
// An order-preserving image of x, never 0: -0 counts as +0, a NaN as the
// largest value.
__device__ __forceinline__ uint32_t image(float x) {
  if (x != x) return kNanImage;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float from_image(uint32_t i) {
  if (i == kNanImage) return __int_as_float(0x7fffffff);
  return __uint_as_float((i & 0x80000000u) ? (i & 0x7fffffffu) : ~i);
}
// Value and index as one key: a larger value first, then a lower index.
__device__ __forceinline__ u64 key_of(float x, int index) {
  return (static_cast<u64>(image(x)) << 32) | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ int index_of(u64 key) { return static_cast<int>(~static_cast<uint32_t>(key)); }

// Sums over a part of a row relative to 2^r; r = -inf and s = 0 for nothing.
struct Stats {
  float r, s, w;
};

__device__ __forceinline__ float clamped(float y) { return y < -1e4f ? -1e4f : y; }  // keeps a NaN

// The same sums relative to r >= a.r.
__device__ __forceinline__ void raise(Stats& a, float r) {
  if (a.s != 0.f) {  // true for a NaN
    const float d = clamped(a.r - r), f = ex2_approx(d);
    a.w = f * fmaf(d, a.s, a.w);
    a.s *= f;
  }
  a.r = r;
}
__device__ __forceinline__ Stats merge(Stats a, Stats b) {
  const float r = fmaxf(a.r, b.r);
  raise(a, r);
  raise(b, r);
  return {r, a.s + b.s, a.w + b.w};
}
// A reference for x, whose y passes a's: ceil(x c), and where that product's
// rounding says too little by whole numbers (from 2^24 on; an exponential could
// pass the largest float from 2^32 on), what the rounding left, rounded up.
__device__ __forceinline__ void raise_for(Stats& a, float x, float c) {
  float r = ceilf(x * c);
  const float over = fmaf(x, c, -r);
  if (over > 0.5f) r = __fadd_ru(r, over);
  raise(a, r);
}
// One value of at least -1e30, or NaN, under a reference >= x c.
__device__ __forceinline__ void take(Stats& a, float x, float c) {
  const float y = fmaf(x, c, -a.r), e = ex2_approx(y);
  a.s += e;
  a.w = fmaf(e, y, a.w);
}
constexpr float kFar = 4194304.f;  // 2^22: up to here R is a whole number within 2 of the largest y
constexpr float kLow = -1e29f;

template <int W>
__device__ __forceinline__ void group_sync() {
  if (W == 1)
    __syncwarp();
  else
    __syncthreads();
}

constexpr int kMaxTop = SB_LOGPROBS_MAX_TOP;

struct FwdArgs {
  const void* x;
  long ld;
  int rows, v;
  float c;      // log2(e) / temperature
  float inv_t;  // 1 / temperature
  const float* targets;
  float* logp;
  float* entropy;
  float* lse;
  int k;
  int* top_ids;
  float* top_logp;
};

template <int W>
struct alignas(16) RowShared {
  static constexpr int kCap = W == 1 ? 384 : 1024;
  u64 cand[kCap];
  unsigned short again[W * 32];  // threads whose values are looked at again
  u64 best[kMaxTop];
  u64 group[W == 1 ? 32 : 64];  // the groups' bounds
  u64 bound;
  Stats part[W];
  Stats all;
  int count, threads;
};

// W warps a row (1, 4 or 8) or a part of one (16, CLUSTER); rows of a block: 8
// with W = 1, else 1. In a cluster
// of C blocks each takes 1 / C of the row and rank 0 joins the parts.
template <typename T, int W, bool CLUSTER>
__global__ void __launch_bounds__(W == 1 ? 256 : W * 32, W == 1 ? 6 : 40 / W) logprobs_kernel(FwdArgs a) {
  constexpr int E = Elem<T>::N;
  constexpr int NT = W * 32;
  constexpr int U = 4;  // vectors in flight per thread
  using RS = RowShared<W>;
  __shared__ RS shared_rows[W == 1 ? 8 : 1];
  const int slot = W == 1 ? threadIdx.x / 32 : 0;
  RS& sh = shared_rows[slot];
  const int tid = W == 1 ? threadIdx.x % 32 : threadIdx.x, lane = threadIdx.x % 32, warp = tid / 32;
  int rank = 0, ranks = 1;
  int row;
  if (CLUSTER) {
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    row = blockIdx.x / ranks;
  } else {
    row = W == 1 ? blockIdx.x * 8 + slot : blockIdx.x;
  }
  pdl_wait();
  if (W == 1 && row >= a.rows) return;  // whole warps; nothing below joins warps

  const T* x = static_cast<const T*>(a.x) + static_cast<long>(row) * a.ld;
  // [0, head) and [head + nvec * E, v) singly, the rest in aligned vectors
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int head = min(a.v, off ? E - off : 0);
  const int nvec = (a.v - head) / E;
  const int tail0 = head + nvec * E;
  const int v0 = static_cast<int>(static_cast<long>(nvec) * rank / ranks);
  const int v1 = static_cast<int>(static_cast<long>(nvec) * (rank + 1) / ranks);
  const int loose = rank == 0 ? head + (a.v - tail0) : 0;  // single values, of rank 0
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  const auto loose_at = [&](int i) { return i < head ? i : tail0 + (i - head); };
  const float c = a.c;

  Stats st{kNegInf, 0.f, 0.f};
  float best = kNegInf;  // this thread's largest vector: its maximum and place
  int best_vec = -1;
  for (int i0 = v0 + tid; i0 < v1; i0 += U * NT) {
    uint4 u[U];
    float hi[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (i0 + j * NT < v1) u[j] = __ldg(xv + i0 + j * NT);
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = i0 + j * NT;
      hi[j] = i < v1 ? Elem<T>::most(u[j]) : kNegInf;
      if (i < v1 && (hi[j] > best || best_vec < 0)) {
        best = hi[j];
        best_vec = i;
      }
    }
    float top = hi[0];
#pragma unroll
    for (int j = 1; j < U; ++j) top = max_nan(top, hi[j]);
    if (top < kLow) continue;
    if (fmaf(top, c, -st.r) > 0.f) raise_for(st, top, c);
    const float2 r2 = make_float2(-st.r, -st.r), c2 = make_float2(c, c);
    float2 s2 = make_float2(st.s, 0.f), w2 = make_float2(st.w, 0.f);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (i0 + j * NT < v1) {
        float f[E];
        Elem<T>::unpack(Elem<T>::floored(u[j]), f);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 y = __ffma2_rn(make_float2(f[e], f[e + 1]), c2, r2);
          const float2 q = make_float2(ex2_approx(y.x), ex2_approx(y.y));
          s2 = __fadd2_rn(s2, q);
          w2 = __ffma2_rn(q, y, w2);
        }
      }
    }
    st.s = s2.x + s2.y;
    st.w = w2.x + w2.y;
  }
  if (tid < loose) {
    const float f = Elem<T>::get(x + loose_at(tid));
    if (!(f < kLow)) {
      if (fmaf(f, c, -st.r) > 0.f) raise_for(st, f, c);
      take(st, f, c);
    }
  }

  // the row's statistics, in a fixed order
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Stats b{__shfl_xor_sync(0xffffffffu, st.r, o), __shfl_xor_sync(0xffffffffu, st.s, o),
                  __shfl_xor_sync(0xffffffffu, st.w, o)};
    st = merge(st, b);
  }
  if (W == 1) {
    if (lane == 0) sh.all = st;
  } else {
    if (lane == 0) sh.part[warp] = st;
    __syncthreads();
    if (warp == 0) {
      Stats t = lane < W ? sh.part[lane] : Stats{kNegInf, 0.f, 0.f};
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const Stats b{__shfl_xor_sync(0xffffffffu, t.r, o), __shfl_xor_sync(0xffffffffu, t.s, o),
                      __shfl_xor_sync(0xffffffffu, t.w, o)};
        t = merge(t, b);
      }
      if (lane == 0) sh.all = t;
    }
  }

  if (a.k > 0) {
    // lower bounds of the threads' best logits (the last place of the vector),
    // and this thread's upper bound (its first place)
    const bool any = best_vec >= 0;
    const int first = head + best_vec * E;
    const u64 upper = any ? key_of(best, first) : 0;
    const u64 lower = any ? key_of(best, first + E - 1) : 0;
    constexpr int G = W == 1 ? 32 : 64, PER = NT / G;
    u64 mine = lower;
#pragma unroll
    for (int o = PER / 2; o > 0; o >>= 1) {
      const u64 other = __shfl_xor_sync(0xffffffffu, mine, o);
      mine = other > mine ? other : mine;
    }
    if (tid % PER == 0) sh.group[tid / PER] = mine;
    if (tid == 0) sh.count = sh.threads = 0;
    group_sync<W>();
    if (tid < G) {
      // of equal keys, which only groups without a vector have, the first
      const u64 key = sh.group[tid];
      int above = 0;
#pragma unroll 16
      for (int j = 0; j < G; ++j) {
        const u64 o = sh.group[j];
        above += o > key || (o == key && j < tid);
      }
      if (above == a.k - 1) sh.bound = key;
    }
    group_sync<W>();
    // a NaN hides from the maxima: with one in the row every logit is looked at
    const bool odd = sh.all.s != sh.all.s;
    const u64 bound = odd ? 0 : sh.bound;
    const auto offer = [&](float f, int i) {
      const u64 key = key_of(f, i);
      if (key >= bound) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < RS::kCap) sh.cand[at] = key;
      }
    };
    if (any && (odd || upper >= bound)) sh.again[atomicAdd(&sh.threads, 1)] = tid;
    group_sync<W>();
    {
      // the vectors of those threads, dealt out to all
      const int each = (v1 - v0 + NT - 1) / NT, all = sh.threads * each;
#pragma unroll 2
      for (int q = tid; q < all; q += NT) {
        const int i = v0 + sh.again[q / each] + q % each * NT;
        if (i >= v1) continue;
        const uint4 u = __ldg(xv + i);
        if (!odd && key_of(Elem<T>::most(u), head + i * E) < bound) continue;
        float f[E];
        Elem<T>::unpack(u, f);
#pragma unroll
        for (int e = 0; e < E; ++e) offer(f[e], head + i * E + e);
      }
    }
    if (tid < loose) offer(Elem<T>::get(x + loose_at(tid)), loose_at(tid));
    group_sync<W>();
    const int n = sh.count;
    if (n <= RS::kCap) {
      // each candidate's place is the number of larger ones (keys differ)
      for (int i = tid; i < n; i += NT) {
        const u64 mine = sh.cand[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += sh.cand[j] > mine;
        if (above < a.k) sh.best[above] = mine;
      }
      if (tid < a.k && tid >= n) sh.best[tid] = 0;
    } else {
      // more candidates than places (sorted or equal logits): the best key
      // below the last one, k times over the row
      u64 last = ~0ull;
      for (int t = 0; t < a.k; ++t) {
        u64 b = 0;
        for (int i = v0 + tid; i < v1; i += NT) {
          float f[E];
          Elem<T>::unpack(__ldg(xv + i), f);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const u64 key = key_of(f[e], head + i * E + e);
            if (key < last && key > b) b = key;
          }
        }
        if (tid < loose) {
          const u64 key = key_of(Elem<T>::get(x + loose_at(tid)), loose_at(tid));
          if (key < last && key > b) b = key;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const u64 other = __shfl_xor_sync(0xffffffffu, b, o);
          b = other > b ? other : b;
        }
        if (W > 1) {
          if (lane == 0) sh.group[warp] = b;
          __syncthreads();
          b = 0;
          for (int j = 0; j < W; ++j) b = sh.group[j] > b ? sh.group[j] : b;
          __syncthreads();
        }
        if (tid == 0) sh.best[t] = b;
        last = b;
      }
    }
  }

  Stats all;
  if (CLUSTER) {
    cluster_sync();
    if (rank != 0) {
      cluster_sync();  // rank 0 reads this block's shared memory until then
      return;
    }
    const uint32_t all_addr = smem_u32(&sh.all), best_addr = smem_u32(&sh.best[0]);
    all = Stats{kNegInf, 0.f, 0.f};
    for (int r = 0; r < ranks; ++r) {
      Stats b;
      const uint32_t at = mapa_shared(all_addr, r);
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.r) : "r"(at));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.s) : "r"(at + 4));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.w) : "r"(at + 8));
      all = merge(all, b);
    }
    if (a.k > 0) {
      const int n = ranks * a.k;
      for (int i = tid; i < n; i += NT) {
        u64 key;
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key) : "r"(mapa_shared(best_addr, i / a.k) + (i % a.k) * 8));
        sh.cand[i] = key;
      }
      __syncthreads();
      cluster_sync();
      for (int i = tid; i < n; i += NT) {
        const u64 mine = sh.cand[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += sh.cand[j] > mine;
        if (mine != 0 && above < a.k) sh.best[above] = mine;
      }
      __syncthreads();
    } else {
      cluster_sync();
    }
  } else {
    group_sync<W>();
    all = sh.all;
  }

  // Nothing above -1e29, or a reference too far out: the sums again, by
  // differences to the largest logit, over the whole row.
  float ref = 0.f;  // what is taken off the logits first
  const bool low = all.s == 0.f || (all.s == all.s && fabsf(all.r) > kFar);
  if (low) {
    float m = kNegInf;
    for (int i = tid; i < a.v; i += NT) m = fmaxf(m, Elem<T>::get(x + i));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (W > 1) {
      __syncthreads();
      if (lane == 0) sh.part[warp].r = m;
      __syncthreads();
      for (int i = 0; i < W; ++i) m = fmaxf(m, sh.part[i].r);
      __syncthreads();
    }
    ref = m;
    Stats t{m == kNegInf ? kNegInf : 0.f, 0.f, 0.f};
    if (m != kNegInf)
      for (int i = tid; i < a.v; i += NT) take(t, fmaxf(Elem<T>::get(x + i) - m, -1e30f), c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      t.s += __shfl_xor_sync(0xffffffffu, t.s, o);
      t.w += __shfl_xor_sync(0xffffffffu, t.w, o);
    }
    if (W > 1) {
      if (lane == 0) sh.part[warp] = t;
      __syncthreads();
      t.s = t.w = 0.f;
      for (int i = 0; i < W; ++i) {
        t.s += sh.part[i].s;
        t.w += sh.part[i].w;
      }
    }
    all = t;
  }
  const float log_s = log2f(all.s);  // log2 of the sum relative to 2^r
  const bool none = all.s == 0.f;
  // log probability of a logit: none for -inf (and NaN in a row with a NaN)
  const auto logp_of = [&](float f) {
    if (all.s != all.s) return all.s;
    if (f == kNegInf) return kNegInf;
    if (low) return fmaf(f - ref, a.inv_t, -log_s * kLn2);  // in log2 units it might pass the largest float
    return (fmaf(f, c, -all.r) - log_s) * kLn2;
  };
  if (tid == 0) {
    // ref / temperature and r + log2 S, the first 0 unless the row was taken again
    if (a.lse) a.lse[row] = all.s != all.s ? all.s : (none ? kNegInf : fmaf(ref, a.inv_t, (all.r + log_s) * kLn2));
    if (a.entropy) a.entropy[row] = none ? 0.f : (log_s - all.w / all.s) * kLn2;
    if (a.logp) {
      const float t = a.targets[row];
      const int i = static_cast<int>(t);
      const bool known = static_cast<float>(i) == t && i >= 0 && i < a.v;
      a.logp[row] = known ? logp_of(Elem<T>::get(x + i)) : 0.f;
    }
  }
  if (tid < a.k) {
    const u64 key = sh.best[tid];
    const long at = static_cast<long>(row) * a.k + tid;
    if (a.top_ids) a.top_ids[at] = index_of(key);
    if (a.top_logp) a.top_logp[at] = logp_of(from_image(static_cast<uint32_t>(key >> 32)));
  }
}

// dx_j = (g (1[j = t] - p_j) - h p_j (log p_j + H)) / temperature, elementwise
// given lse and H; g counts only for a given token that exists.
struct BwdArgs {
  const void* x;
  long ld;
  int rows, v;
  float inv_t;     // 1 / temperature
  float c, c_lo;   // log2(e) / temperature as the sum of two floats
  const float* targets;
  const float* lse;
  const float* entropy;
  const float* dlogp;
  const float* dentropy;
  void* dx;
  long ldd;
  int chunks;  // blocks per row
};

struct RowGrad {
  float l2, l2_lo;  // lse in log2 units, and what its rounding left
  float c, c_lo;    // log2(e) / temperature, likewise
  float g, h;       // dlogp, dentropy, over temperature
  float gh;         // -(g + h H); NaN where lse is
  float hl;         // -h ln2
  int t;            // given token or -1
};

// ex2.approx with subnormal results: p of 2^-126 and less still counts where
// its factor is large.
__device__ __forceinline__ float ex2_full(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The part of dx that all logits have, -(g p + h p (log p + H)). log2 p is
// kept in [-1e4, 0]: -inf stays a number, and where the rounding of a large
// lse says p > 1, p = 1.
template <bool ACCURATE>
__device__ __forceinline__ float grad_of(float x, const RowGrad& r) {
  float y = fmaf(x, r.c, -r.l2);
  if (ACCURATE && y > -1e4f) y += fmaf(x, r.c_lo, -r.l2_lo);
  y = fminf(fmaxf(y, -1e4f), 0.f);
  return ex2_full(y) * fmaf(r.hl, y, r.gh);
}

template <typename T>
__global__ void __launch_bounds__(256) logprobs_bwd_kernel(BwdArgs a) {
  constexpr int E = Elem<T>::N;
  constexpr bool kAccurate = sizeof(T) == 4;
  pdl_wait();
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  const T* x = static_cast<const T*>(a.x) + static_cast<long>(row) * a.ld;
  T* dx = static_cast<T*>(a.dx) + static_cast<long>(row) * a.ldd;
  RowGrad r;
  const float lse = a.lse[row];
  constexpr float kLog2eLo = 1.9259630e-8f;  // log2(e) - kLog2e
  r.l2 = lse * kLog2e;
  r.l2_lo = fmaf(lse, kLog2eLo, fmaf(lse, kLog2e, -r.l2));
  r.c = a.c;
  r.c_lo = a.c_lo;
  const float t = a.dlogp ? a.targets[row] : -1.f;
  const int ti = static_cast<int>(t);
  r.t = (static_cast<float>(ti) == t && ti >= 0 && ti < a.v) ? ti : -1;
  r.g = r.t >= 0 ? a.dlogp[row] * a.inv_t : 0.f;
  r.h = a.dentropy ? a.dentropy[row] * a.inv_t : 0.f;
  r.gh = a.dentropy ? -fmaf(r.h, a.entropy[row], r.g) : -r.g;
  r.hl = -r.h * kLn2;
  if (lse == kNegInf) r.g = r.gh = r.hl = 0.f;
  if (lse != lse) r.gh = lse;
  const auto value = [&](float f, int j) { return grad_of<kAccurate>(f, r) + (j == r.t ? r.g : 0.f); };
  const auto put = [&](int j, float d) {
    if (sizeof(T) == 4)
      reinterpret_cast<float*>(dx)[j] = d;
    else
      reinterpret_cast<__nv_bfloat16*>(dx)[j] = __float2bfloat16_rn(d);
  };

  const uintptr_t xa = reinterpret_cast<uintptr_t>(x) & 15, da = reinterpret_cast<uintptr_t>(dx) & 15;
  if (xa != da) {  // rows that start at different places of a vector
    for (int j = chunk * 256 + threadIdx.x; j < a.v; j += a.chunks * 256) put(j, value(Elem<T>::get(x + j), j));
    return;
  }
  const int off = static_cast<int>(xa / sizeof(T));
  const int head = min(a.v, off ? E - off : 0);
  const int nvec = (a.v - head) / E, tail0 = head + nvec * E;
  if (chunk == 0) {
    const int loose = head + (a.v - tail0);
    if (threadIdx.x < loose) {
      const int j = threadIdx.x < head ? threadIdx.x : tail0 + (threadIdx.x - head);
      put(j, value(Elem<T>::get(x + j), j));
    }
  }
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  uint4* dv = reinterpret_cast<uint4*>(dx + head);
  constexpr int U = 4;
  for (int i0 = chunk * 256 * U + threadIdx.x; i0 < nvec; i0 += a.chunks * 256 * U) {
    uint4 u[U];
#pragma unroll
    for (int q = 0; q < U; ++q)
      if (i0 + q * 256 < nvec) u[q] = xv[i0 + q * 256];
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int i = i0 + q * 256;
      if (i >= nvec) break;
      float f[E];
      Elem<T>::unpack(u[q], f);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = grad_of<kAccurate>(f[e], r);
      const unsigned at = static_cast<unsigned>(r.t - (head + i * E));
      if (at < static_cast<unsigned>(E)) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (at == static_cast<unsigned>(e)) f[e] += r.g;
      }
      uint4 o;
      if (sizeof(T) == 4)
        o = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
      else
        o = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4 % E], f[5 % E]),
                       pack_bf16x2(f[6 % E], f[7 % E]));
      dv[i] = o;
    }
  }
}

// A warp, 4 or 8 a row.
template <typename T, int W>
int launch_rows(const FwdArgs& a, cudaStream_t s) {
  const int blocks = W == 1 ? (a.rows - 1) / 8 + 1 : a.rows;
  logprobs_kernel<T, W, false><<<blocks, W == 1 ? 256 : W * 32, 0, s>>>(a);
  return cudaPeekAtLastError() == cudaSuccess ? 0 : SB_OPERR_LAUNCH;
}
// A row cut over a cluster of blocks of 16 warps.
template <typename T>
int launch_cut(const FwdArgs& a, int cluster, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows) * cluster);
  cfg.blockDim = dim3(512);
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, logprobs_kernel<T, 16, true>, a) == cudaSuccess ? 0 : SB_OPERR_LAUNCH;
}

template <typename T>
int fwd_t(const FwdArgs& a, cudaStream_t s) {
  // A warp, 4 or 8 a row: more than the row's length pays for wait longer for
  // one another (8192 rows of 4000 bf16: 30 us with a warp, 40 with 4; of 16000:
  // 109, 76 and 101 with 8; of 128256, 4096 rows: 250 with 4, 204 with 8). Rows
  // that cannot fill the SMs are cut over a cluster, up to 8 blocks of at least
  // 512 vectors a row.
  const int nvec = a.v / Elem<T>::N;
  if (nvec <= 512) return launch_rows<T, 1>(a, s);
  int cluster = 1;
  while (cluster < 8 && static_cast<long>(a.rows) * cluster * 2 <= 2L * num_sms_cached() && nvec / (2 * cluster) >= 512)
    cluster *= 2;
  if (cluster > 1) return launch_cut<T>(a, cluster, s);
  return nvec <= 4096 ? launch_rows<T, 4>(a, s) : launch_rows<T, 8>(a, s);
}

}  // namespace

int token_logprobs(const LogprobsDesc& d, cudaStream_t s) {
  if (d.rows == 0) return 0;
  FwdArgs a;
  a.x = d.x;
  a.ld = d.ld;
  a.rows = d.rows;
  a.v = d.v;
  a.inv_t = 1.0f / d.temperature;
  a.c = static_cast<float>(1.4426950408889634074 / static_cast<double>(d.temperature));
  a.targets = d.targets;
  a.logp = d.logp;
  a.entropy = d.entropy;
  a.lse = d.lse;
  a.k = d.k;
  a.top_ids = d.top_ids;
  a.top_logp = d.top_logp;
  return d.f32 ? fwd_t<float>(a, s) : fwd_t<__nv_bfloat16>(a, s);
}

int token_logprobs_bwd(const LogprobsBwdDesc& d, cudaStream_t s) {
  if (d.rows == 0) return 0;
  BwdArgs a;
  a.x = d.x;
  a.ld = d.ld;
  a.rows = d.rows;
  a.v = d.v;
  a.inv_t = 1.0f / d.temperature;
  const double c = 1.4426950408889634074 / static_cast<double>(d.temperature);
  a.c = static_cast<float>(c);
  a.c_lo = static_cast<float>(c - static_cast<double>(a.c));
  a.targets = d.targets;
  a.lse = d.lse;
  a.entropy = d.entropy;
  a.dlogp = d.dlogp;
  a.dentropy = d.dentropy;
  a.dx = d.dx;
  a.ldd = d.ldd;
  const int per_block = 256 * 4 * (d.f32 ? 4 : 8);  // one round of a block's vectors
  a.chunks = std::max(1, (d.v + per_block - 1) / per_block);
  const long blocks = static_cast<long>(d.rows) * a.chunks;
  if (blocks > 0x7fffffffL) return SB_OPERR_ARGS;
  if (d.f32)
    logprobs_bwd_kernel<float><<<static_cast<unsigned>(blocks), 256, 0, s>>>(a);
  else
    logprobs_bwd_kernel<__nv_bfloat16><<<static_cast<unsigned>(blocks), 256, 0, s>>>(a);
  return cudaPeekAtLastError() == cudaSuccess ? 0 : SB_OPERR_LAUNCH;
}

}  // namespace sb
