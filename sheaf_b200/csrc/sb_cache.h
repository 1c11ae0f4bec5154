// Host launch interface of cached generation: the paged key/value cache, the
// attention over it, and the scoring of tokens (internal to the library).
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "../../include/sheaf_b200_ops.h"

namespace sb {

// Error-word code of an index (page, position) outside what it indexes: the
// kernel skips the access and records this (sb_op_device_error).
constexpr int kErrIndex = 2;
// (It does not take the place of a timeout, which is the graver news.)
__device__ __forceinline__ void report_index(int* err) {
  if (err) atomicCAS(err, 0, kErrIndex);
}

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

struct AppendDesc {
  sb_kv_cache cache;
  const void* qkv;
  int64_t ld;
  int n, h_q;
  void* q_out;
  int64_t ldq;
  const int32_t* seq;
  const int32_t* pos;
  int base;
  const int32_t* pages;
  int n_seqs, max_pages;
  int rotary, rot_dim;
  const float* cos;
  const float* sin;
  int n_pos;
};
int kv_append(const AppendDesc& d, cudaStream_t s, int* err);

struct PrefixAttnDesc {
  sb_kv_cache cache;
  const void* q;
  int64_t ldq;
  void* out;
  int64_t ldo;
  float* lse;  // [b * tq, h_q] or null
  int b, tq, h_q;
  float scale;
  const int32_t* prefix_pages;
  int prefix_len;
  const int32_t* pages;
  int max_pages;
  const int32_t* lens;
};
size_t prefix_attention_workspace_bytes(const PrefixAttnDesc& d);
int prefix_attention(const PrefixAttnDesc& d, void* ws, size_t ws_bytes, cudaStream_t s, int* err);

struct LogprobsDesc {
  bool f32;
  const void* x;
  int64_t ld;
  int rows, v;
  const float* targets;
  float temperature;
  float* logp;
  float* entropy;
  float* lse;
  int k;
  int32_t* top_ids;
  float* top_logp;
};
int token_logprobs(const LogprobsDesc& d, cudaStream_t s);

struct LogprobsBwdDesc {
  bool f32;
  const void* x;
  int64_t ld;
  int rows, v;
  const float* targets;
  float temperature;
  const float* lse;
  const float* entropy;
  const float* dlogp;
  const float* dentropy;
  void* dx;
  int64_t ldd;
};
int token_logprobs_bwd(const LogprobsBwdDesc& d, cudaStream_t s);

}  // namespace sb
