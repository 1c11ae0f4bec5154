// Log probabilities of given tokens, the entropy of their distributions, the
// most likely alternatives, and the VJP.
//
// With z = x / temperature, a row of v logits, t its given token:
//   lse = log sum_j exp z_j      logp = z_t - lse
//   H   = - sum_j p_j log p_j    p = exp(z - lse)
// One pass keeps, per thread, the largest logit m, S = sum 2^y and
// W = sum 2^y y with y = (x - m) log2(e) / temperature, so that
//   lse = m / temperature + ln2 log2 S,   H = ln2 (log2 S - W / S):
// the entropy comes from differences to m and keeps its relative accuracy
// when one token has nearly all the probability.
//
// The k best (larger value first, then lower index) come from the same pass:
// each thread remembers its largest 16-byte vector. The k-th largest of 32
// groups of threads bounds the k-th best logit from below, so only threads
// whose own best reaches that bound look at their part of the row again
// (from L2), and only logits that reach it become candidates.
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

// The largest logit of a part of a row, and sums over it relative to that.
struct Stats {
  float m, s, w;
};

__device__ __forceinline__ float clamped(float y) { return y < -1e4f ? -1e4f : y; }  // keeps a NaN

__device__ __forceinline__ void raise(Stats& a, float m, float c) {
  if (a.s != 0.f) {  // true for a NaN
    const float d = clamped((a.m - m) * c), f = ex2_approx(d);
    a.w = f * (a.w + d * a.s);
    a.s *= f;
  }
  a.m = m;
}
__device__ __forceinline__ Stats merge(Stats a, Stats b, float c) {
  const float m = fmaxf(a.m, b.m);
  raise(a, m, c);
  raise(b, m, c);
  return {m, a.s + b.s, a.w + b.w};
}
// One value under a.m >= x; -inf has no probability.
__device__ __forceinline__ void take(Stats& a, float x, float c) {
  if (x == kNegInf) return;
  const float y = clamped((x - a.m) * c), e = ex2_approx(y);
  a.s += e;
  a.w = fmaf(e, y, a.w);
}

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
  static constexpr int kCap = W == 1 ? 192 : 1024;
  u64 cand[kCap];
  u64 best[kMaxTop];
  u64 lane_key[32];
  u64 bound;
  Stats part[W];
  Stats all;
  int count;
};

// W warps per row part; rows of a block: 8 with W = 1, else 1. In a cluster
// of C blocks each takes 1 / C of the row and rank 0 joins the parts.
template <typename T, int W, bool CLUSTER>
__global__ void __launch_bounds__(W == 1 ? 256 : W * 32, W == 1 ? 6 : 48 / W) logprobs_kernel(FwdArgs a) {
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
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (i0 + j * NT < v1) u[j] = __ldg(xv + i0 + j * NT);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = i0 + j * NT;
      if (i >= v1) break;
      float f[E];
      Elem<T>::unpack(u[j], f);
      float hi = f[0], lo = f[0];
#pragma unroll
      for (int e = 1; e < E; ++e) {
        hi = fmaxf(hi, f[e]);
        lo = fminf(lo, f[e]);
      }
      if (hi > best || best_vec < 0) {
        best = hi;
        best_vec = i;
      }
      if (lo >= -1e30f && hi <= 1e30f && st.m != kNegInf) {
        if (hi > st.m) raise(st, hi, c);
        const float2 m2 = make_float2(-st.m, -st.m), c2 = make_float2(c, c);
        float2 s2 = make_float2(st.s, 0.f), w2 = make_float2(st.w, 0.f);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 y = __fmul2_rn(__fadd2_rn(make_float2(f[e], f[e + 1]), m2), c2);
          const float2 q = make_float2(ex2_approx(y.x), ex2_approx(y.y));
          s2 = __fadd2_rn(s2, q);
          w2 = __ffma2_rn(q, y, w2);
        }
        st.s = s2.x + s2.y;
        st.w = w2.x + w2.y;
      } else {
        if (hi > st.m) raise(st, hi, c);
#pragma unroll
        for (int e = 0; e < E; ++e) take(st, f[e], c);
      }
    }
  }
  if (tid < loose) {
    const float f = Elem<T>::get(x + loose_at(tid));
    if (f > st.m) raise(st, f, c);
    take(st, f, c);
  }

  // the row's statistics, in a fixed order
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Stats b{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
                  __shfl_xor_sync(0xffffffffu, st.w, o)};
    st = merge(st, b, c);
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
        const Stats b{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.s, o),
                      __shfl_xor_sync(0xffffffffu, t.w, o)};
        t = merge(t, b, c);
      }
      if (lane == 0) sh.all = t;
    }
  }

  if (a.k > 0) {
    // lower bounds of the groups' best logits (the last place of the vector),
    // and this thread's upper bound (its first place)
    const bool any = best_vec >= 0;
    const int first = head + best_vec * E;
    const u64 upper = any ? key_of(best, first) : 0;
    const u64 lower = any ? key_of(best, first + E - 1) : 0;
    if (W == 1) {
      sh.lane_key[lane] = lower;
    } else {
      // group = 2 W threads of one or neighbouring warps: W groups of 32
      // threads each when W = 32; here 32 groups of NT / 32 = W threads
      u64 g = lower;
#pragma unroll
      for (int o = W / 2; o > 0; o >>= 1) {
        const u64 other = __shfl_xor_sync(0xffffffffu, g, o);
        g = other > g ? other : g;
      }
      if (tid % W == 0) sh.lane_key[tid / W] = g;
    }
    if (tid == 0) sh.count = 0;
    group_sync<W>();
    if (warp == 0) {
      const u64 mine = sh.lane_key[lane];
      int above = 0;
      for (int j = 0; j < 32; ++j) {
        const u64 o = sh.lane_key[j];
        above += (o > mine) || (o == mine && j < lane);
      }
      if (above == a.k - 1) sh.bound = mine;
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
    if (odd || (any && upper >= bound)) {
      for (int i = v0 + tid; i < v1; i += NT) {
        float f[E];
        Elem<T>::unpack(__ldg(xv + i), f);
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
          if (lane == 0) sh.lane_key[warp] = b;
          __syncthreads();
          b = 0;
          for (int j = 0; j < W; ++j) b = sh.lane_key[j] > b ? sh.lane_key[j] : b;
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
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.m) : "r"(at));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.s) : "r"(at + 4));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.w) : "r"(at + 8));
      all = merge(all, b, c);
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

  const float log_s = log2f(all.s);  // log2 of the sum relative to the maximum
  const bool none = all.m == kNegInf && all.s == 0.f;
  // log probability of a logit: none for -inf (and NaN in a row with a NaN)
  const auto logp_of = [&](float f) {
    if (all.s != all.s) return all.s;
    if (f == kNegInf) return kNegInf;
    return ((f - all.m) * c - log_s) * kLn2;
  };
  if (tid == 0) {
    if (a.lse) a.lse[row] = all.s != all.s ? all.s : (none ? kNegInf : fmaf(all.m, a.inv_t, log_s * kLn2));
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

template <typename T, int W>
int launch_fwd(const FwdArgs& a, int cluster, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.blockDim = dim3(W == 1 ? 256 : W * 32);
  cfg.stream = s;
  cudaError_t e;
  if (cluster > 1) {
    cfg.gridDim = dim3(static_cast<unsigned>(a.rows) * cluster);
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, logprobs_kernel<T, W == 1 ? 16 : W, true>, a);
  } else {
    cfg.gridDim = dim3(W == 1 ? (a.rows + 7) / 8 : a.rows);
    e = cudaLaunchKernelEx(&cfg, logprobs_kernel<T, W, false>, a);
  }
  return e == cudaSuccess ? 0 : SB_OPERR_LAUNCH;
}

template <typename T>
int fwd_t(const FwdArgs& a, cudaStream_t s) {
  // Rows that cannot fill the SMs are cut over a cluster: up to 8 blocks of
  // at least 1024 vectors a row.
  const int nvec = a.v / Elem<T>::N;
  if (nvec <= 256) return launch_fwd<T, 1>(a, 1, s);
  int cluster = 1;
  while (cluster < 8 && static_cast<long>(a.rows) * cluster * 2 <= 2L * num_sms_cached() && nvec / (2 * cluster) >= 512)
    cluster *= 2;
  if (cluster > 1) return launch_fwd<T, 16>(a, cluster, s);
  if (nvec <= 1024) return launch_fwd<T, 4>(a, 1, s);
  return launch_fwd<T, 16>(a, 1, s);
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
