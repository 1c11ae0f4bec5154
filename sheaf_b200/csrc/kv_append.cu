// Appending new tokens' keys and values to a paged cache, with the rotation
// of queries and keys by their positions done on the way.
//
// Token i of sequence s at position p goes to page pages[s][(p - base) / R],
// row (p - base) % R of the cache (R rows a page). Queries and keys turn by
// the angles of row p of the cos / sin tables, pair by pair:
//   (a, b) -> (a cos - b sin, b cos + a sin)
// in float32, rounded once to the element type; values are copied.
//
// A thread owns one unit of a token's heads: two vectors of 16 bytes that
// hold whole pairs (for the halves layout a vector and its partner rot / 2
// further on), for HPT heads, so that the angles are read once for HPT
// heads and 2 HPT loads are in flight. Moving the bytes bounds it: 16384 tokens
// of 32 + 8 + 8 heads of 128 in bf16, 403 MB, take 62 us at the measured copy
// rate; 69 without rotation, 78 with pairs, 83 with halves (two heads a thread,
// four blocks an SM; one head 101, four heads 99); float32 126, 0.97 of the
// rate. The angles' 64 bytes a thread, from L1, are what bf16 pays for.
#include <cuda_bf16.h>

#include <algorithm>

#include "sb_cache.h"
#include "sb_kernels.h"
#define SB_PDL_FAMILY 1
#include "sb_launch.cuh"

namespace sb {

namespace {

enum : int { kRotNone = SB_ROTARY_NONE, kRotHalves = SB_ROTARY_HALVES, kRotPairs = SB_ROTARY_PAIRS };

// (No more than 16-byte alignment: what the entry point and the dispatch below
// see to. Eight angles are two vectors.)
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) Pack {
  T v[VEC];
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float& d, float x) { d = x; }
__device__ __forceinline__ void from_f32(__nv_bfloat16& d, float x) { d = __float2bfloat16_rn(x); }

// (a, b) turned by (c, n) = (cos, sin). Which product of a sum is rounded first
// is spelt out, for each type as its vector path always had it, so that a value
// comes out the same whichever path its alignment leads to.
template <typename T>
__device__ __forceinline__ float2 turned(float a, float b, float c, float n) {
  const float x = fmaf(a, c, -__fmul_rn(b, n));
  return make_float2(x, sizeof(T) == 4 ? fmaf(a, n, __fmul_rn(b, c)) : fmaf(b, c, __fmul_rn(a, n)));
}

template <typename T>
struct AppendArgs {
  T* k;
  T* v;
  long page_stride, row_stride, head_stride;
  int n_pages, hkv, hd;
  FastDiv page_rows;
  FastDiv units, per_token;  // units of a head; threads of a token
  const T* qkv;
  long ld;
  int n, hq;
  T* q_out;
  long ldq;
  const int* seq;
  const int* pos;
  int base;
  const int* pages;
  int n_seqs, max_pages;
  int rot;
  const float* cos;
  const float* sin;
  int n_pos;
  int* err;
};

template <typename T, int VEC, int MODE, int HPT>
__global__ void __launch_bounds__(256, 4) kv_append_kernel(AppendArgs<T> a) {
  using P = Pack<T, VEC>;
  const int heads = a.hq + 2 * a.hkv;
  const uint32_t idx = blockIdx.x * blockDim.x + threadIdx.x;
  const uint32_t t = a.per_token(idx);
  if (t >= static_cast<uint32_t>(a.n)) return;
  const long token = t;
  const uint32_t rest = idx - t * a.per_token.d, group = a.units(rest);
  const int h0 = group * HPT, u = rest - group * a.units.d;

  // element offsets of the unit's two vectors within a head
  const int half = a.rot / 2;
  int e0, e1;
  bool turns = false;
  if (MODE == kRotHalves && u < half / VEC) {
    e0 = u * VEC;
    e1 = e0 + half;
    turns = true;
  } else {
    e0 = 2 * u * VEC;
    e1 = e0 + VEC;
    if (MODE == kRotPairs) turns = e0 < a.rot;
  }

  P x[HPT][2];
  const T* src = a.qkv + token * a.ld;
#pragma unroll
  for (int i = 0; i < HPT; ++i)
    if (h0 + i < heads) {
      x[i][0] = *reinterpret_cast<const P*>(src + static_cast<long>(h0 + i) * a.hd + e0);
      x[i][1] = *reinterpret_cast<const P*>(src + static_cast<long>(h0 + i) * a.hd + e1);
    }

  const int s = a.seq[token], p = a.pos[token];
  bool live = s >= 0;  // a negative sequence marks a padding token
  if (live && (s >= a.n_seqs || p < a.base || (MODE != kRotNone && p >= a.n_pos) ||
               static_cast<int>(a.page_rows(p - a.base)) >= a.max_pages)) {
    live = false;
    report_index(a.err);
  }
  long row = -1;  // element offset of the token's row in the cache
  if (live) {
    const int own = p - a.base, nth = a.page_rows(own), page = a.pages[static_cast<long>(s) * a.max_pages + nth];
    if (page >= 0 && page < a.n_pages)
      row = page * a.page_stride + static_cast<long>(own - nth * static_cast<int>(a.page_rows.d)) * a.row_stride;
    else
      report_index(a.err);
  }

  if (MODE != kRotNone && live && h0 < a.hq + a.hkv) {
    const float* ct = a.cos + static_cast<long>(p) * half;
    const float* st = a.sin + static_cast<long>(p) * half;
    if (MODE == kRotHalves || VEC == 1) {
      if (turns) {
        const int j = MODE == kRotHalves ? e0 : e0 / 2;
        const Pack<float, VEC> c = *reinterpret_cast<const Pack<float, VEC>*>(ct + j);
        const Pack<float, VEC> n = *reinterpret_cast<const Pack<float, VEC>*>(st + j);
#pragma unroll
        for (int i = 0; i < HPT; ++i)
          if (h0 + i < a.hq + a.hkv)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const float2 y = turned<T>(to_f32(x[i][0].v[e]), to_f32(x[i][1].v[e]), c.v[e], n.v[e]);
              from_f32(x[i][0].v[e], y.x);
              from_f32(x[i][1].v[e], y.y);
            }
      }
    } else {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int e = w ? e1 : e0;
        if (e >= a.rot) continue;
        constexpr int HV = VEC > 1 ? VEC / 2 : 1;
        const Pack<float, HV> c = *reinterpret_cast<const Pack<float, HV>*>(ct + e / 2);
        const Pack<float, HV> n = *reinterpret_cast<const Pack<float, HV>*>(st + e / 2);
#pragma unroll
        for (int i = 0; i < HPT; ++i)
          if (h0 + i < a.hq + a.hkv)
#pragma unroll
            for (int j = 0; j < HV; ++j) {
              const float2 y = turned<T>(to_f32(x[i][w].v[2 * j]), to_f32(x[i][w].v[(2 * j + 1) % VEC]), c.v[j], n.v[j]);
              from_f32(x[i][w].v[2 * j], y.x);
              from_f32(x[i][w].v[(2 * j + 1) % VEC], y.y);
            }
      }
    }
  }

#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = h0 + i;
    if (h >= heads) break;
    T* dst;
    if (h < a.hq) {
      if (!live) x[i][0] = x[i][1] = P{};  // a padding token's query row is zero
      dst = a.q_out + token * a.ldq + static_cast<long>(h) * a.hd;
    } else {
      if (row < 0) continue;
      const int kh = h - a.hq;
      dst = kh < a.hkv ? a.k + row + kh * a.head_stride : a.v + row + (kh - a.hkv) * a.head_stride;
    }
    *reinterpret_cast<P*>(dst + e0) = x[i][0];
    *reinterpret_cast<P*>(dst + e1) = x[i][1];
  }
}

template <typename T, int VEC, int MODE, int HPT>
int launch(AppendArgs<T> a, cudaStream_t s) {
  const int groups = (a.hq + 2 * a.hkv + HPT - 1) / HPT, units = a.hd / (2 * VEC);
  a.units = FastDiv::of(units);
  a.per_token = FastDiv::of(groups * units);
  // threads are counted in 31 bits: more tokens than that take several launches
  const int most = std::max(1, 0x7fff0000 / (groups * units)), n = a.n;
  for (int at = 0; at < n; at += std::min(most, n - at)) {
    AppendArgs<T> part = a;
    part.n = std::min(most, n - at);
    part.qkv += at * a.ld;
    part.q_out += a.hq ? at * a.ldq : 0;
    part.seq += at;
    part.pos += at;
    const unsigned blocks = (static_cast<unsigned>(part.n) * (groups * units) + 255) / 256;
    kv_append_kernel<T, VEC, MODE, HPT><<<blocks, 256, 0, s>>>(part);
  }
  return cudaPeekAtLastError() == cudaSuccess ? 0 : SB_OPERR_LAUNCH;
}

template <typename T, int VEC, int HPT>
int by_mode(const AppendArgs<T>& a, int mode, cudaStream_t s) {
  if (mode == kRotHalves) return launch<T, VEC, kRotHalves, HPT>(a, s);
  if (mode == kRotPairs) return launch<T, VEC, kRotPairs, HPT>(a, s);
  return launch<T, VEC, kRotNone, HPT>(a, s);
}

template <typename T>
int append_t(const AppendDesc& d, cudaStream_t s, int* err) {
  AppendArgs<T> a;
  a.k = static_cast<T*>(d.cache.k);
  a.v = static_cast<T*>(d.cache.v);
  a.page_stride = d.cache.page_stride;
  a.row_stride = d.cache.row_stride;
  a.head_stride = d.cache.head_stride;
  a.n_pages = d.cache.n_pages;
  a.page_rows = FastDiv::of(d.cache.page_rows);
  a.hkv = d.cache.n_heads;
  a.hd = d.cache.head_dim;
  a.qkv = static_cast<const T*>(d.qkv);
  a.ld = d.ld;
  a.n = d.n;
  a.hq = d.h_q;
  a.q_out = static_cast<T*>(d.q_out);
  a.ldq = d.ldq;
  a.seq = d.seq;
  a.pos = d.pos;
  a.base = d.base;
  a.pages = d.pages;
  a.n_seqs = d.n_seqs;
  a.max_pages = d.max_pages;
  a.rot = d.rotary == kRotNone ? 0 : d.rot_dim;
  a.cos = d.cos;
  a.sin = d.sin;
  a.n_pos = d.n_pos;
  a.err = err;
  constexpr int VEC = 16 / sizeof(T);
  const auto aligned = [](const void* p, long stride) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * sizeof(T) % 16 == 0;
  };
  const auto table = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  bool vec = aligned(d.qkv, d.ld) && (!d.q_out || aligned(d.q_out, d.ldq));
  // whole units of pairs, and angle rows that start on 16 bytes
  if (a.rot) vec = vec && a.rot % (2 * VEC) == 0 && a.rot % 8 == 0 && table(d.cos) && table(d.sin);
  if (!vec) return by_mode<T, 1, 1>(a, d.rotary, s);
  return by_mode<T, VEC, 2>(a, d.rotary, s);
}

}  // namespace

int kv_append(const AppendDesc& d, cudaStream_t s, int* err) {
  if (d.n == 0) return 0;
  return d.cache.elem == SB_ELEM_F32 ? append_t<float>(d, s, err) : append_t<__nv_bfloat16>(d, s, err);
}

}  // namespace sb
