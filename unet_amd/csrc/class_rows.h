// Shared pieces of the kernels over class logits (class_probs.hip, distill.hip).
//
// A "row" is one prediction over C classes.  Row r = o * inner + i (o < outer, i < inner); its logit of class c lies at
// element o*so + i*si + c*sc: [N][C] rows have inner = 1 and sc = 1, class maps [B][C][H][W] have inner = H*W, si = 1
// and sc = H*W.  What belongs to a row with k entries (top alternatives, a teacher's slots) lies at [o][k][i].
//
// With m = max x, c2 = log2(e) / T:  s = sum 2^((x - m) c2), L2 = log2 s, p = 2^((x - m) c2 - L2).  Statistics are fp32
// whatever the logits' type; the difference x - m is taken before the product, so that logits of the size of the
// type's lowest value (masks) neither overflow nor cancel.
//   row without a finite logit: m = 0, L2 = +inf, hence p = 0 everywhere;
//   row with a NaN or +inf:     L2 = NaN, hence p = NaN everywhere.
#pragma once
#include "common.h"
#include <math.h>

typedef _Float16 f16;

struct RowView {
  long long outer, inner, so, si, sc;
  int C;
  __device__ __forceinline__ long long base(long long r) const {
    if (inner == 1) return r * so;
    const long long o = r / inner;
    return o * so + (r - o * inner) * si;
  }
  // element of entry k of row r in a dense [outer][K][inner] table
  __device__ __forceinline__ long long entry(long long r, int k, int K) const {
    if (inner == 1) return r * K + k;
    const long long o = r / inner;
    return (o * K + k) * inner + (r - o * inner);
  }
};

static inline RowView uh_row_view(const uh_class_view* v) { return RowView{v->outer, v->inner, v->so, v->si, v->sc, v->classes}; }

// what every entry point checks of a view; rows are counted in 31 bits so that a launch can cover them
static inline int uh_check_view(const uh_class_view* v, const char* who) {
  UH_REQUIRE(v, "%s: no view", who);
  UH_REQUIRE(v->dtype >= UH_F32 && v->dtype <= UH_F16, "%s: dtype %d", who, v->dtype);
  UH_REQUIRE(v->classes > 0 && v->classes <= UH_CLASSES_MAX, "%s: %d classes (1 to %d)", who, v->classes, UH_CLASSES_MAX);
  UH_REQUIRE(v->outer > 0 && v->inner > 0 && v->outer <= 0x7fffffffll && v->inner <= 0x7fffffffll &&
                 v->outer * v->inner <= 0x7fffffffll,
             "%s: %lld x %lld rows (1 to 2^31 - 1)", who, v->outer, v->inner);
  UH_REQUIRE(v->so >= 0 && v->si >= 0 && v->sc >= 0, "%s: negative stride", who);
  return UH_OK;
}

template <typename T> __device__ __forceinline__ float ld(const T* p) { return (float)*p; }
__device__ __forceinline__ void st(float* p, float v) { *p = v; }
__device__ __forceinline__ void st(bf16* p, float v) { *p = (bf16)v; }
__device__ __forceinline__ void st(f16* p, float v) { *p = (f16)v; }      // overflow gives inf, which a GradScaler looks for

static constexpr float UH_LN2 = 0.693147180559945309f;
static constexpr float UH_LOG2E = 1.44269504088896341f;
static constexpr float UH_ZMIN = -200.f;      // 2^-200 is 0 in fp32: below it a term of the entropy sum is 0

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// (x - m) / T of a reported value; x - m may overflow where its quotient does not (a class masked with the type's lowest
// value, T > 1)
__device__ __forceinline__ float scaled(float x, float m, float temperature) {
  const float d = x - m;
  return d == -INFINITY ? x / temperature - m / temperature : d / temperature;
}

// order[x] as unsigned: larger logits first, -0 = +0; the low half orders equal logits by class, lowest first.
// 0 stands for "none": masked classes (-inf) are never alternatives.
__device__ __forceinline__ uint32_t order32(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unorder32(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
__device__ __forceinline__ uint64_t rank_key(float x, int c) {
  return x > -INFINITY ? ((uint64_t)order32(x) << 32) | (uint32_t)~c : 0ull;
}
__device__ __forceinline__ int key_class(uint64_t k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float key_value(uint64_t k) { return unorder32((uint32_t)(k >> 32)); }

template <int G> __device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
template <int G> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <int G> __device__ __forceinline__ uint64_t group_max(uint64_t v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    const uint64_t w = ((uint64_t)__shfl_xor((uint32_t)(v >> 32), o, 64) << 32) | __shfl_xor((uint32_t)v, o, 64);
    v = v > w ? v : w;
  }
  return v;
}

// over a workgroup of 256 threads; `buf` has 4 entries and may be reused after the call
template <typename V> __device__ __forceinline__ V block_max(V v, V* buf) {
  v = group_max<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  v = buf[0];
#pragma unroll
  for (int w = 1; w < 4; ++w) v = v > buf[w] ? v : buf[w];
  return v;
}
__device__ __forceinline__ float block_sum(float v, float* buf) {
  v = group_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  return (buf[0] + buf[1]) + (buf[2] + buf[3]);
}

__device__ __forceinline__ long long load_int(const void* p, int bytes, long long i) {
  return bytes == 8 ? ((const long long*)p)[i] : (long long)((const int*)p)[i];
}

// statistics of one row by a workgroup of 256 threads: m, s and t = sum e z2 (for the entropy)
struct RowStat { float m, s, t; };
template <typename T> __device__ RowStat block_row_stat(const T* __restrict__ x, int C, long long sc, float c2, float* buf) {
  float m = -INFINITY;
  for (int c = threadIdx.x; c < C; c += 256) m = fmaxf(m, ld(x + c * sc));
  m = block_max(m, buf);
  if (m == -INFINITY) m = 0.f;
  float s = 0.f, t = 0.f;
  for (int c = threadIdx.x; c < C; c += 256) {
    const float z = (ld(x + c * sc) - m) * c2, e = ex2(z);
    s += e;
    t = fmaf(e, fmaxf(z, UH_ZMIN), t);
  }
  s = block_sum(s, buf);
  t = block_sum(t, buf);
  return RowStat{m, s, t};
}
__device__ __forceinline__ float stat_l2(float s) { return s == 0.f ? INFINITY : log2f(s); }
