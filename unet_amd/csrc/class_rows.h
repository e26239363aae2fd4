// Shared pieces of the kernels over class logits (class_probs.hip, distill.hip).
//
// A "row" is one prediction over C classes.  Row r = o * inner + i (o < outer, i < inner); its logit of class c lies at
// element o*so + i*si + c*sc: [N][C] rows have inner = 1 and sc = 1, class maps [B][C][H][W] have inner = H*W, si = 1
// and sc = H*W.  What belongs to a row with k entries (top alternatives, a teacher's slots) lies at [o][k][i].
//
// Statistics of a row, fp32 whatever the logits' type: m = max x, and with c = log2(e) / T, M = c m rounded to fp32
//     s = sum 2^(c x - M),   t = sum 2^(c x - M) (c x - M)          one fused multiply-add and one exponential each
// The rounding of M, r = c m - M, is a common factor 2^r of s that ln s = log(s) - r ln 2 takes out again.  It is at most 1/2 for
// |M| < 2^24, where it costs less than the sums' own roundings, and grows with |M|: past 2^31 2^r itself would overflow or vanish.
//   |M| >= 2^24 ("far": rows masked throughout with -1e9 or the type's lowest value, very small temperatures): 2^(c (x - m))
//     instead, an instruction more an element, with s and t relative to m itself (r = 0);
//   a row without a finite logit: m = 0, s = 0, and p = 0 everywhere;  a row with a NaN or +inf: s = NaN.
//
// Which kernel takes a row (uh_class_path below): rows whose classes lie side by side are read by a group of lanes, 16 bytes
// a load, and stay in registers between the maximum, the sums and the gradient; up to 64 classes, or classes that lie apart
// (maps), a row is one thread's; anything else is one workgroup's, element by element.
#pragma once
#include "common.h"
#include <math.h>

typedef _Float16 f16;

struct RowView {
  long long inner, so, si, sc;    // inner = 1 where one step walks all rows, whatever the tensor's shape
  long long einner;               // the view's own inner: what has k entries per row is laid out by it
  int C;
  __device__ __forceinline__ long long base(long long r) const {
    if (inner == 1) return r * so;
    const unsigned o = (unsigned)r / (unsigned)inner;             // rows are counted in 31 bits
    return o * so + ((unsigned)r - o * (unsigned)inner) * si;
  }
  // element of entry k of row r in a dense [outer][K][inner] table
  __device__ __forceinline__ long long entry(long long r, int k, int K) const {
    if (einner == 1) return r * K + k;
    const unsigned o = (unsigned)r / (unsigned)einner;
    return ((long long)o * K + k) * einner + ((unsigned)r - o * (unsigned)einner);
  }
};

static inline RowView uh_row_view(const uh_class_view* v) {
  RowView w{v->inner, v->so, v->si, v->sc, v->inner, v->classes};
  if (w.inner > 1 && (v->outer == 1 || w.so == w.inner * w.si)) {
    w.so = w.si;
    w.inner = 1;
  }
  return w;
}

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

// The range in which c and 1/T are normal numbers with room to spare: products with a logit's difference may overflow, which
// is an exponential of 0.
static inline bool uh_temperature(float t) { return t >= 1e-6f && t <= 1e6f; }

// ---- values -------------------------------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float ld(const T* p) { return (float)*p; }
template <typename T> __device__ __forceinline__ void st(T* p, float v) { *p = (T)v; }   // fp16: overflow gives inf, which a GradScaler looks for

static constexpr float UH_LN2 = 0.693147180559945309f;
static constexpr float UH_ZMIN = -200.f;      // 2^-200 is 0 in fp32: below it a term of t is 0

// v_exp_f32, v_log_f32, v_rcp_f32: good to a unit in the last place, results below the smallest normal number are 0
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float lg2(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ float rcp(float x) { return __builtin_amdgcn_rcpf(x); }

// a maximum whose M is too large for its rounding to be taken out again (c2: log2(e) / T)
__device__ __forceinline__ bool is_far(float m, float c2) { return fabsf(m * c2) >= 0x1p24f; }
struct RowRef {           // the point and the scale a row's exponents are taken in, its maximum not far
  float c, M;
  __device__ __forceinline__ RowRef(float c_, float M_, int) : c(c_), M(M_) {}
  __device__ __forceinline__ RowRef(float m, float c2) : c(c2), M(m * c2) {}
  __device__ __forceinline__ float z(float x) const { return fmaf(x, c, -M); }
  __device__ __forceinline__ float ln_s(float m, float s) const { return (lg2(s) - fmaf(m, c, -M)) * UH_LN2; }
};
struct FarRef {           // the same for one that is
  float c, m;
  __device__ __forceinline__ FarRef(float m_, float c2) : c(c2), m(m_) {}
  __device__ __forceinline__ float z(float x) const { return (x - m) * c; }
};
struct AnyRef {           // either, for a few values: the bits of the other two
  float c, M, sub;
  __device__ __forceinline__ AnyRef(float m, float c2) : c(c2), M(is_far(m, c2) ? 0.f : m * c2), sub(is_far(m, c2) ? m : 0.f) {}
  __device__ __forceinline__ float z(float x) const { return fmaf(x - sub, c, -M); }
  __device__ __forceinline__ float ln_s(float m, float s) const { return (lg2(s) - fmaf(m - sub, c, -M)) * UH_LN2; }
};
// f, a sweep over a row, with the reference that its maximum needs: two copies of the sweep, of which rows of ordinary logits never
// pay for the second.  Lanes of one row agree.
template <typename F> __device__ __forceinline__ void with_ref(float m, float c2, F f) {
  if (__builtin_expect(is_far(m, c2), 0)) f(FarRef(m, c2));
  else f(RowRef(m, c2));
}
// the same for the whole wave, whose rows may differ
template <typename F> __device__ __forceinline__ void with_wave_ref(float m, float c2, F f) {
  if (__builtin_expect(__any(is_far(m, c2)), 0)) f(AnyRef(m, c2));
  else f(RowRef(m, c2));
}
struct RowStat { float m, s, t; };

// (x - m) / T of a reported value; x - m may overflow where its quotient does not (a class masked with the type's lowest
// value, T > 1).  Fused, since m / T may overflow as well: beside x = -inf that would be a NaN.
__device__ __forceinline__ float scaled(float x, float m, float inv_t) {
  const float d = x - m;
  return d == -INFINITY ? fmaf(-m, inv_t, x * inv_t) : d * inv_t;
}

// The exponent that takes sums relative to the point of the maximum m0 to that of m >= m0.
__device__ __forceinline__ float ref_step(float m0, float m, float c2) {
  const bool f0 = is_far(m0, c2), f = is_far(m, c2);
  if (m0 == m) return 0.f;
  return f ? (f0 ? (m0 - m) * c2 : -fmaf(m, c2, -(m0 * c2))) : (f0 ? fmaf(m0, c2, -(m * c2)) : m0 * c2 - m * c2);
}
// joins the statistics of two parts of a row; a part without a finite logit (s = 0) has no say in m
__device__ __forceinline__ RowStat join(const RowStat& a, const RowStat& b, float c2) {
  const float ma = a.s == 0.f ? -INFINITY : a.m, mb = b.s == 0.f ? -INFINITY : b.m;
  float m = fmaxf(ma, mb);
  if (m == -INFINITY) m = 0.f;
  float da = a.m * c2 - m * c2, db = b.m * c2 - m * c2;
  if (__builtin_expect(__any(is_far(a.m, c2) || is_far(b.m, c2)), 0)) da = ref_step(a.m, m, c2), db = ref_step(b.m, m, c2);
  if (a.s == 0.f) da = 0.f;
  if (b.s == 0.f) db = 0.f;
  const float ea = ex2(da), eb = ex2(db);
  RowStat o;
  o.m = m;
  o.s = a.s * ea + b.s * eb;
  o.t = ea * fmaf(a.s, fmaxf(da, UH_ZMIN), a.t) + eb * fmaf(b.s, fmaxf(db, UH_ZMIN), b.t);
  return o;
}

// rank keys: larger logits first, -0 = +0, equal logits by class, lowest first.  0 stands for "none": classes masked with
// -inf are never alternatives.
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

// ---- reductions -----------------------------------------------------------------------------------------------------------
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
// max of three in one instruction; NaNs lose against numbers, as in fmaxf
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}
// over groups of 16 or 64 lanes, result in all of them: rotations inside rows of 16 lanes (0x120 + n), then across rows
template <int G> __device__ __forceinline__ float group_max(float v) {
  v = fmaxf(v, dpp<0x128>(v));
  v = fmaxf(v, dpp<0x124>(v));
  v = fmaxf(v, dpp<0x122>(v));
  v = fmaxf(v, dpp<0x121>(v));
  if (G > 16) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    v = fmaxf(v, __shfl_xor(v, 32, 64));
  }
  return v;
}
template <int G> __device__ __forceinline__ float group_sum(float v) {
  v += dpp<0x128>(v);
  v += dpp<0x124>(v);
  v += dpp<0x122>(v);
  v += dpp<0x121>(v);
  if (G > 16) {
    v += __shfl_xor(v, 16, 64);
    v += __shfl_xor(v, 32, 64);
  }
  return v;
}
template <int G> __device__ __forceinline__ uint64_t group_max(uint64_t v) {
#pragma unroll
  for (int o = (G > 64 ? 64 : G) / 2; o > 0; o >>= 1) {
    const uint64_t w = ((uint64_t)__shfl_xor((uint32_t)(v >> 32), o, 64) << 32) | __shfl_xor((uint32_t)v, o, 64);
    v = v > w ? v : w;
  }
  return v;
}
template <int G> __device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    const uint32_t w = __shfl_xor(v, o, 64);
    v = v > w ? v : w;
  }
  return v;
}

// The wave of a workgroup that does what one wave does alone: another one from workgroup to workgroup, so that this work is
// spread over the four SIMDs of a CU (a wave's number in its workgroup decides its SIMD).
template <int G> __device__ __forceinline__ bool serial_wave() { return G <= 64 || (threadIdx.x >> 6) == ((blockIdx.x + blockIdx.y) & (G / 64 - 1)); }

// LDS of the reductions over a workgroup of NW waves; nothing for groups inside a wave
template <int NW> struct RedBuf {
  float m[NW], s[NW], t[NW];
  uint64_t k[NW];
};
template <> struct RedBuf<0> {};

// over all G lanes of a group (G > 64: the whole workgroup, which must call together)
template <int G> struct Red {
  static constexpr int NW = G > 64 ? G / 64 : 0;
  typedef RedBuf<NW> Buf;
  __device__ static __forceinline__ float max_(float v, Buf& b) {
    v = group_max<(G > 64 ? 64 : G)>(v);
    if constexpr (NW > 0) {
      __syncthreads();
      if ((threadIdx.x & 63) == 0) b.m[threadIdx.x >> 6] = v;
      __syncthreads();
      v = b.m[0];
#pragma unroll
      for (int w = 1; w < NW; ++w) v = fmaxf(v, b.m[w]);
    }
    return v;
  }
  __device__ static __forceinline__ float sum_(float v, Buf& b) {
    v = group_sum<(G > 64 ? 64 : G)>(v);
    if constexpr (NW > 0) {
      __syncthreads();
      if ((threadIdx.x & 63) == 0) b.s[threadIdx.x >> 6] = v;
      __syncthreads();
      v = b.s[0];
#pragma unroll
      for (int w = 1; w < NW; ++w) v += b.s[w];
    }
    return v;
  }
  __device__ static __forceinline__ void sum2(float& v, float& u, Buf& b) {
    v = group_sum<(G > 64 ? 64 : G)>(v);
    u = group_sum<(G > 64 ? 64 : G)>(u);
    if constexpr (NW > 0) {
      __syncthreads();
      if ((threadIdx.x & 63) == 0) { b.s[threadIdx.x >> 6] = v; b.t[threadIdx.x >> 6] = u; }
      __syncthreads();
      v = b.s[0], u = b.t[0];
#pragma unroll
      for (int w = 1; w < NW; ++w) { v += b.s[w]; u += b.t[w]; }
    }
  }
  __device__ static __forceinline__ uint64_t maxkey(uint64_t v, Buf& b) {
    v = group_max<(G > 64 ? 64 : G)>(v);
    if constexpr (NW > 0) {
      __syncthreads();
      if ((threadIdx.x & 63) == 0) b.k[threadIdx.x >> 6] = v;
      __syncthreads();
      v = b.k[0];
#pragma unroll
      for (int w = 1; w < NW; ++w) v = v > b.k[w] ? v : b.k[w];
    }
    return v;
  }
};

__device__ __forceinline__ long long load_int(const void* p, int bytes, long long i) {
  return bytes == 8 ? ((const long long*)p)[i] : (long long)((const int*)p)[i];
}

// Keeps the compiler from working out every `c < C` of an unrolled sweep ahead of it, or from
// keeping them for the next (two scalar registers each, spilled to vector registers).
__device__ __forceinline__ int renew_uniform(int C) {
  C = __builtin_amdgcn_readfirstlane(C);
  asm volatile("" : "+s"(C));
  return C;
}

// ---- a row in the registers of a group of lanes ------------------------------------------------------------------------------
// 16 bytes wherever an element may lie: rows of odd sizes start anywhere (the hardware takes element-aligned vectors).  A vector
// type, whose accesses the compiler takes to meet those of any other type: a class is read and written again by itself through
// float* and the like.  Spelt out for each size, since an alignment that depends on a template's argument is dropped without a word
// (and 16 bytes assumed).
typedef uint32_t LooseVec2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t LooseVec4 __attribute__((ext_vector_type(4), aligned(4)));
template <int BYTES> struct LooseVecOf { typedef LooseVec2 type; };
template <> struct LooseVecOf<4> { typedef LooseVec4 type; };
template <typename T> using LooseVec = typename LooseVecOf<sizeof(T)>::type;
typedef uint32_t Vec16 __attribute__((ext_vector_type(4)));          // on 16 bytes: LDS

// Between stores of one lane and those of another lane of the same wave to the same places: they leave in the order of the program.
__device__ __forceinline__ void wave_stores_in_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

struct Online {
  float top, M, s0, s1, t;
  __device__ __forceinline__ Online() : top(-INFINITY), M(-0x1p24f), s0(0.f), s1(0.f), t(0.f) {}
};

template <typename T, int G, int NV> struct RowRegs {
  static constexpr int E = 16 / sizeof(T);
  static constexpr int CAP = G * NV * E;
  uint32_t w[NV][4];

  __device__ __forceinline__ static uint32_t neg_inf() {
    return sizeof(T) == 4 ? 0xff800000u : std_is_half() ? 0xfc00fc00u : 0xff80ff80u;
  }
  __device__ __forceinline__ static constexpr bool std_is_half() { return __is_same(T, f16); }

  // vector v = r*G + lane holds elements first(v) .. first(v) + E - 1; the last one of a row that is no multiple of E is
  // read so that it ends with the row, with -inf in the places that its left neighbour holds too.  n >= E.
  __device__ __forceinline__ static int first(int r, int lane, int n) {
    const int e = (r * G + lane) * E;
    return e + E <= n ? e : n - E;
  }
  template <bool ONCE> __device__ __forceinline__ void fetch(int r, const char* p) {
    const LooseVec<T>* q = reinterpret_cast<const LooseVec<T>*>(p);
    const LooseVec<T> u = ONCE ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[r][i] = u[i];
  }
  // elements c0 .. c0 + n of the row at p (the same for all lanes of a wave where G >= 64: one scalar address, and an offset of
  // 32 bits a vector); n >= E or c0 >= E
  template <bool ONCE = false> __device__ __forceinline__ void load(const T* __restrict__ p, int c0, int n, int lane) {
    const uint32_t off = (uint32_t)(c0 + lane * E) * (uint32_t)sizeof(T);
    n = renew_uniform(n);
#pragma unroll
    for (int r = 0; r < NV; ++r)
      if ((r + 1) * G * E <= n) {
        fetch<ONCE>(r, (const char*)p + r * G * 16 + (size_t)off);
      } else if (r * G * E < n) {
        if ((r * G + lane) * E < n) fetch<ONCE>(r, (const char*)p + (size_t)((uint32_t)(c0 + first(r, lane, n)) * (uint32_t)sizeof(T)));
        else {
#pragma unroll
          for (int i = 0; i < 4; ++i) w[r][i] = neg_inf();
        }
      }
    // the ragged vector
    if (n % E) {
      const int dup = E - n % E;                                   // places that the left neighbour holds
#pragma unroll
      for (int r = 0; r < NV; ++r)
        if (r * G * E < n && (r + 1) * G * E > n - E) {
          const int e = (r * G + lane) * E;
          if (e < n && e + E > n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (sizeof(T) == 4) {
                if (i < dup) w[r][i] = neg_inf();
              } else {
                if (2 * i < dup) w[r][i] = (w[r][i] & 0xffff0000u) | (neg_inf() & 0xffffu);
                if (2 * i + 1 < dup) w[r][i] = (w[r][i] & 0xffffu) | (neg_inf() & 0xffff0000u);
              }
            }
          }
        }
    }
  }
  // Between two sweeps: without it the compiler unpacks 16-bit logits once and keeps them in twice the registers (256 and
  // spills where 64 hold the row).
  __device__ __forceinline__ void fresh() {
#pragma unroll
    for (int r = 0; r < NV; ++r) asm volatile("" : "+v"(w[r][0]), "+v"(w[r][1]), "+v"(w[r][2]), "+v"(w[r][3]));
  }
  __device__ __forceinline__ float get(int r, int j) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[r][j]);
    else if constexpr (std_is_half()) {
      float v;                                             // the compiler would keep every upper half in a register of its own
      if (j & 1) asm("v_cvt_f32_f16_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:WORD_1" : "=v"(v) : "v"(w[r][j >> 1]));
      else asm("v_cvt_f32_f16 %0, %1" : "=v"(v) : "v"(w[r][j >> 1]));
      return v;
    } else
      return __uint_as_float(j & 1 ? w[r][j >> 1] & 0xffff0000u : w[r][j >> 1] << 16);
  }
  // the largest element, and (NM = NV) that of every vector
  template <int NM = 0> __device__ __forceinline__ float lane_max(int n, float* vmax = nullptr) const {
    float m = -INFINITY;
    n = renew_uniform(n);
#pragma unroll
    for (int r = 0; r < NV; ++r)
      if (r * G * E < n) {
        if constexpr (NM > 0) {
          float v = fmaxf(get(r, 0), get(r, 1));
#pragma unroll
          for (int j = 2; j < E; j += 2) v = max3(v, get(r, j), get(r, j + 1));
          vmax[r] = v;
          m = fmaxf(m, v);
        } else {
#pragma unroll
          for (int j = 0; j < E; j += 2) m = max3(m, get(r, j), get(r, j + 1));
        }
        __builtin_amdgcn_sched_barrier(0);                  // one vector at a time: unpacked ones would pile up
      }
    return m;
  }
  // s and (ENT) t of a lane's elements, even and odd ones apart.  Without CLAMP a class of -inf makes t a NaN; the -inf that
  // fill the row's last vectors do not.
  template <bool ENT, bool CLAMP = false, typename R> __device__ __forceinline__ void add_sums(const R& ref, int n, float& s0, float& s1, float& t0, float& t1) const {
    n = renew_uniform(n);
#pragma unroll
    for (int r = 0; r < NV; ++r)
      if (r * G * E < n) {
        if (!ENT || CLAMP || (r + 1) * G * E <= n) add_vector<ENT, ENT && CLAMP>(r, ref, s0, s1, t0, t1);
        else add_vector<ENT, ENT>(r, ref, s0, s1, t0, t1);
        __builtin_amdgcn_sched_barrier(0);
      }
  }
  template <bool ENT, bool CLAMP, typename R> __device__ __forceinline__ void add_vector(int r, const R& ref, float& s0, float& s1, float& t0, float& t1) const {
#pragma unroll
    for (int j = 0; j < E; j += 2) {
      const float z0 = ref.z(get(r, j)), z1 = ref.z(get(r, j + 1));
      const float e0 = ex2(z0), e1 = ex2(z1);
      s0 += e0, s1 += e1;
      if (ENT) t0 = fmaf(e0, CLAMP ? fmaxf(z0, UH_ZMIN) : z0, t0), t1 = fmaf(e1, CLAMP ? fmaxf(z1, UH_ZMIN) : z1, t1);
    }
  }
  template <bool ENT, bool CLAMP = false, typename R> __device__ __forceinline__ void lane_sums(const R& ref, int n, float& s, float& t) const {
    float s0 = 0.f, s1 = 0.f, t0 = 0.f, t1 = 0.f;
    add_sums<ENT, CLAMP>(ref, n, s0, s1, t0, t1);
    s = s0 + s1, t = t0 + t1;
  }
  // Largest element, s and (ENT) t of a lane in one sweep that takes the vectors as they arrive: against the running maximum's
  // M, not below -2^24 (a row whose maximum is not far loses nothing by it), which is returned; a vector that raises it rescales
  // what is summed.  vmax as in lane_max.
  template <bool ENT, int NM> __device__ __forceinline__ void online(float c2, int n, Online& o, float* vmax) const {
    n = renew_uniform(n);
#pragma unroll
    for (int r = 0; r < NV; ++r)
      if (r * G * E < n) {
        float v = online_vector<ENT>(r, c2, ENT && (r + 1) * G * E > n, o);
        if (NM > 0) vmax[r] = v;
        __builtin_amdgcn_sched_barrier(0);
      }
  }
  template <bool ENT> __device__ __forceinline__ float online_vector(int r, float c2, bool clamp, Online& o) const {
    float v = fmaxf(get(r, 0), get(r, 1));
#pragma unroll
    for (int j = 2; j < E; j += 2) v = max3(v, get(r, j), get(r, j + 1));
    o.top = fmaxf(o.top, v);
    const float M = fmaxf(o.top * c2, -0x1p24f), d = o.M - M, f = ex2(d);
    if (ENT) o.t = f * fmaf(o.s0 + o.s1, d, o.t);
    o.s0 *= f, o.s1 *= f;
    o.M = M;
    const RowRef ref(c2, M, 0);
    float t1 = 0.f;
    if (clamp) add_vector<ENT, ENT>(r, ref, o.s0, o.s1, o.t, t1);
    else add_vector<ENT, false>(r, ref, o.s0, o.s1, o.t, t1);
    if (ENT) o.t += t1;
    // now: terms left to be summed later would take registers of their own
    if (ENT) asm volatile("" : "+v"(o.s0), "+v"(o.s1), "+v"(o.t), "+v"(o.top));
    else asm volatile("" : "+v"(o.s0), "+v"(o.s1), "+v"(o.top));
    return v;
  }
  // f(x) of every element to out[c0 .. c0 + n)
  template <typename F> __device__ __forceinline__ void map_store(T* __restrict__ out, int c0, int n, int lane, F f) const {
    const uint32_t off = (uint32_t)(c0 + lane * E) * (uint32_t)sizeof(T);
    n = renew_uniform(n);
#pragma unroll
    for (int r = 0; r < NV; ++r) {
      if ((r + 1) * G * E <= n) {
        put(r, (char*)out + r * G * 16 + (size_t)off, f);
      } else if (r * G * E < n) {
        const int e = (r * G + lane) * E;
        if (e + E <= n) put(r, (char*)out + r * G * 16 + (size_t)off, f);
        else if (e < n) {
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (n - E + j >= e) out[c0 + n - E + j] = (T)f(get(r, j));
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  template <typename F> __device__ __forceinline__ void put(int r, char* p, F f) const {
    LooseVec<T> u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) u[i] = __float_as_uint(f(get(r, i)));
      else {
        typedef __attribute__((ext_vector_type(2))) T T2;
        const T2 v = {(T)f(get(r, 2 * i)), (T)f(get(r, 2 * i + 1))};
        u[i] = __builtin_bit_cast(uint32_t, v);
      }
    }
    *reinterpret_cast<LooseVec<T>*>(p) = u;
  }
};

// s and t of a row in registers, given its maximum.  The clamp of its exponents, one instruction of nine an element, is only for
// classes of -inf (0 times -inf): rows that hold one are found by their NaN and summed again with it.
template <typename T, int G, int NV, typename R>
__device__ __forceinline__ void group_sums(RowRegs<T, G, NV>& x, const R& ref, int n, RowStat& s, typename Red<G>::Buf& red) {
  x.template lane_sums<true>(ref, n, s.s, s.t);
  Red<G>::sum2(s.s, s.t, red);
  const bool again = s.t != s.t && s.s == s.s;
  if (G >= 64 ? again : (bool)__any(again)) {
    float s2, t2;
    x.template lane_sums<true, true>(ref, n, s2, t2);
    Red<G>::sum2(s2, t2, red);
    if (again) s.t = t2;
  }
}
// Statistics of a row (or part) in registers of a workgroup, whose loads may still be on their way: the sums are done while they
// arrive, instead of after the last of them, when nothing would be on its way.  lane_top: the lane's largest.
template <typename T, int G, int NV, bool ENT, int NM>
__device__ __forceinline__ RowStat arriving_stat(RowRegs<T, G, NV>& x, float c2, int n, float& lane_top, float* vmax, typename Red<G>::Buf& red) {
  Online o;
  x.template online<ENT, NM>(c2, n, o, vmax);
  lane_top = o.top;
  x.fresh();                                                 // once, ahead of the branches: in them it would copy the row
  RowStat s;
  s.m = Red<G>::max_(o.top, red);
  if (s.m == -INFINITY) s.m = 0.f;
  if (is_far(s.m, c2)) {                                     // what was summed is of no use
    const FarRef far(s.m, c2);
    if (ENT) group_sums<T, G, NV>(x, far, n, s, red);
    else {
      x.template lane_sums<false>(far, n, s.s, s.t);
      s.s = Red<G>::sum_(s.s, red);
    }
    return s;
  }
  const RowRef ref(s.m, c2);
  const float d = o.M - ref.M, f = ex2(d);
  s.s = (o.s0 + o.s1) * f;
  if (ENT) {
    s.t = f * fmaf(o.s0 + o.s1, d, o.t);
    Red<G>::sum2(s.s, s.t, red);
    if (s.t != s.t && s.s == s.s) {                          // a class of -inf
      float s2, t2;
      x.template lane_sums<true, true>(ref, n, s2, t2);
      Red<G>::sum2(s2, t2, red);
      s.t = t2;
    }
  } else {
    s.t = 0.f;
    s.s = Red<G>::sum_(s.s, red);
  }
  return s;
}

// Inside a loop over rows: keeps the compiler from carrying every vector's place in a row from turn to turn (two registers
// a vector, which cost a third of the waves).
__device__ __forceinline__ int renew(int lane) {
  asm volatile("" : "+v"(lane));
  return lane;
}

// statistics of one row by G lanes of a workgroup (any strides, element by element)
template <typename T, int G> __device__ RowStat strided_row_stat(const T* __restrict__ x, int C, long long sc, float c2, int lane,
                                                                 typename Red<G>::Buf& buf) {
  float m = -INFINITY;
  for (int c = lane; c < C; c += G) m = fmaxf(m, ld(x + c * sc));
  m = Red<G>::max_(m, buf);
  if (m == -INFINITY) m = 0.f;
  const AnyRef ref(m, c2);
  float s = 0.f, t = 0.f;
  for (int c = lane; c < C; c += G) {
    const float z = ref.z(ld(x + c * sc)), e = ex2(z);
    s += e;
    t = fmaf(e, fmaxf(z, UH_ZMIN), t);
  }
  Red<G>::sum2(s, t, buf);
  return RowStat{m, s, t};
}

// ---- the largest of a row ---------------------------------------------------------------------------------------------------
// A lane's N largest so far, falling, with their classes (-1: none).  Classes come in rising order, so that a strict
// comparison keeps the lowest of equal ones; x = -inf and NaN never enter.  A value's new place takes the middle of its own,
// its left neighbour's and x: one instruction for the value, a comparison and two selections for the class.
template <int N> struct TopList {
  float v[N];
  int c[N];
  __device__ __forceinline__ TopList() {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = -INFINITY, c[i] = -1;
  }
  __device__ __forceinline__ void insert(float x, int cls) {
#pragma unroll
    for (int i = N - 1; i > 0; --i) {
      const int here = select(x > v[i], cls, c[i]);
      c[i] = select(x > v[i - 1], c[i - 1], here);
      v[i] = __builtin_amdgcn_fmed3f(x, v[i - 1], v[i]);
    }
    c[0] = select(x > v[0], cls, c[0]);
    v[0] = max3(x, v[0], v[0]);
  }
  // a selection that stays one: the compiler makes branches of nested ones
  __device__ __forceinline__ static int select(bool p, int a, int b) {
    int d = p ? a : b;
    asm("" : "+v"(d));
    return d;
  }
  __device__ __forceinline__ void pop() {
#pragma unroll
    for (int i = 0; i + 1 < N; ++i) v[i] = v[i + 1], c[i] = c[i + 1];
    v[N - 1] = -INFINITY, c[N - 1] = -1;
  }
};
// x if it comes behind (v, c) in the order of the alternatives, else -inf
__device__ __forceinline__ float behind(float x, int cls, float v, int c) { return x < v || (x == v && cls > c) ? x : -INFINITY; }

__device__ __forceinline__ int ballot_count(bool p) { return __popcll(__ballot(p)); }

// A lower bound of the k-th largest of a wave's NK keys a lane, with at least k keys at or above it; 0 if there are fewer than k
// keys.  Bit by bit from the highest in which the keys differ down to the 16th: what the lower bits would exclude is a few
// candidates more than k.
template <int NK> __device__ __forceinline__ uint32_t wave_kth(const uint32_t (&key)[NK], int k) {
  uint32_t any = 0, all = ~0u;
  int n = 0;
#pragma unroll
  for (int i = 0; i < NK; ++i) any |= key[i], all &= key[i], n += ballot_count(key[i] != 0);
  if (n < k) return 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) any |= __shfl_xor(any, o, 64), all &= __shfl_xor(all, o, 64);
  const uint32_t differ = any ^ all;
  uint32_t low = differ ? all & ~((2u << (31 - __clz(differ))) - 1u) : all;
  for (int bit = differ ? 31 - __clz(differ) : 0; bit >= 15; --bit) {
    const uint32_t test = low | (1u << bit);
    n = 0;
#pragma unroll
    for (int i = 0; i < NK; ++i) n += ballot_count(key[i] >= test);
    if (n >= k) {
      low = test;
      if (n == k) break;
    }
  }
  return low;
}

// One wave cuts a list of n > k different keys in LDS down to fewer, the k largest among them, and returns how many are left: a
// search for the k-th largest, bit by bit; it ends above the keys' lower halves unless so many values are equal that the classes
// have to decide.  The keys move to the front: a step reads its 64 places before it writes, and no further than it has read.
__device__ __forceinline__ int wave_cut(uint64_t* list, int n, int k) {
  const int lane = threadIdx.x & 63;
  uint64_t low = 0;
  if (n <= 512) {
    uint32_t key[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) key[i] = i * 64 + lane < n ? (uint32_t)(list[i * 64 + lane] >> 32) : 0u;
    low = (uint64_t)wave_kth<8>(key, k) << 32;
  } else if (n <= 1024) {
    uint32_t key[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) key[i] = i * 64 + lane < n ? (uint32_t)(list[i * 64 + lane] >> 32) : 0u;
    low = (uint64_t)wave_kth<16>(key, k) << 32;
  } else {
    int above = n;
    for (int bit = 63; bit >= 0 && (bit >= 47 || above > 2 * k + 128); --bit) {
      const uint64_t test = low | (1ull << bit);
      int c = 0;
      for (int i = lane; i - lane < n; i += 256) {
#pragma unroll
        for (int j = 0; j < 256; j += 64) c += ballot_count(i + j < n && list[i + j] >= test);
      }
      if (c >= k) {
        low = test;
        above = c;
        if (c == k) break;
      }
    }
  }
  int at = 0;
  for (int i = 0; i < n; i += 64) {
    const uint64_t mine = i + lane < n ? list[i + lane] : 0;
    const uint64_t who = __ballot(mine >= low && mine != 0);
    __builtin_amdgcn_wave_barrier();
    if (mine >= low && mine != 0) list[at + __popcll(who & ((1ull << lane) - 1))] = mine;
    __builtin_amdgcn_wave_barrier();
    at += __popcll(who);
  }
  return at;
}
// G lanes: emit(rank, key) of the k largest of n different keys in LDS (16-byte aligned, one place to spare), emit(rank, 0) for
// the places left over.  A key's rank is the number of larger ones, so that the list is cut down first where it is long; of many
// equal values a long one may be left: then all is compared with all.  count: a word of LDS.  Ends with the list still being
// read: the caller's next write to it needs a barrier before.
template <int G, typename F> __device__ __forceinline__ void group_rank(uint64_t* list, int n, int lane, int k, int* count, F emit) {
  if (n > 128 && n > k) {
    if (lane < 64) {
      const int left = wave_cut(list, n, k);
      if (lane == 0) *count = left;
    }
    __syncthreads();
    n = *count;
  }
  if (lane == 0) list[n] = 0;                                // pairs of keys are read
  __syncthreads();
  typedef __attribute__((ext_vector_type(2))) unsigned long long Pair;
  const Pair* pairs = reinterpret_cast<const Pair*>(list);
  for (int i = lane; i < n; i += 2 * G) {
    const bool two = i + G < n;
    const uint64_t a = list[i], b = two ? list[i + G] : ~0ull;
    int ra = 0, rb = 0;
#pragma unroll 4
    for (int j = 0; j < (n + 1) / 2; ++j) {
      const Pair p = pairs[j];
      ra += (p.x > a) + (p.y > a);
      rb += (p.x > b) + (p.y > b);
    }
    if (ra < k) emit(ra, a);
    if (two && rb < k) emit(rb, b);
  }
  for (int i = n + lane; i < k; i += G) emit(i, 0ull);
}

// The k largest of a row in registers.  The k-th largest of the lanes' own maxima bounds the k-th largest element from
// below (each of k lanes holds one at least as large): the few elements at or above it go to a list in LDS.
template <int G> struct TopBuf {
  static constexpr int CAP = G > 64 ? 1024 : 512;
  alignas(16) uint64_t list[CAP + 2];
  float lane_max[G > 64 ? G : 1];
  uint32_t low;
  int count, left;
};
// Fills b.list and returns how many there are (more than CAP: the list is of no use); low: their bound's order32 (0: none).
// All G lanes call; the list stays until the next call.
template <typename T, int G, int NV>
__device__ __forceinline__ int group_candidates(RowRegs<T, G, NV>& x, int n, int lane, int c0, int k, float lane_max, const float* vmax, TopBuf<G>& b,
                                                uint32_t& low) {
  constexpr int E = RowRegs<T, G, NV>::E;
  __syncthreads();                                           // the list of the row before is read no more
  if (lane == 0) b.count = 0;
  const uint32_t mine = lane_max > -INFINITY ? order32(lane_max) : 0u;
  if constexpr (G == 64) {
    const uint32_t key[1] = {mine};
    low = wave_kth<1>(key, k);
  } else {
    b.lane_max[lane] = lane_max;
    __syncthreads();
    if (serial_wave<G>()) {
      uint32_t key[G / 64];
#pragma unroll
      for (int i = 0; i < G / 64; ++i) {
        const float v = b.lane_max[(lane & 63) + 64 * i];
        key[i] = v > -INFINITY ? order32(v) : 0u;
      }
      const uint32_t l = wave_kth<G / 64>(key, k);
      if ((lane & 63) == 0) b.low = l;
    }
    __syncthreads();
    low = b.low;
  }
  const float cut = low ? unorder32(low) : -3.402823466e38f;
  x.fresh();
  n = renew_uniform(n);
  if (__any(mine != 0 && mine >= low)) {                     // one look per vector; its few hits are placed by ballots
#pragma unroll
    for (int r = 0; r < NV; ++r)
      if (r * G * E < n) {
        if (!__any(vmax[r] >= cut)) continue;
        unsigned long long hit[E], some = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) some |= hit[j] = __ballot(x.get(r, j) >= cut);
        if (some) {
          int total = 0, at = 0;
#pragma unroll
          for (int j = 0; j < E; ++j) total += __popcll(hit[j]);
          if ((lane & 63) == 0) at = atomicAdd(&b.count, total);
          at = __builtin_amdgcn_readfirstlane(at);
          const int e = c0 + RowRegs<T, G, NV>::first(r, lane, n);
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (hit[j]) {
              const float v = x.get(r, j);
              const int to = at + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(hit[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hit[j], 0));
              if (v >= cut && to < TopBuf<G>::CAP) b.list[to] = rank_key(v, e + j);
              at += __popcll(hit[j]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
  }
  __syncthreads();
  return b.count;
}
// rows whose many equal values overflow the list: the largest k times over
template <typename T, int G, typename F>
__device__ __forceinline__ void group_rounds(const T* __restrict__ row, int n, int lane, int c0, int k, typename Red<G>::Buf& red, F emit) {
  uint64_t last = ~0ull;
  for (int i = 0; i < k; ++i) {
    uint64_t best = 0;
    for (int c = lane; c < n; c += G) {
      const uint64_t key = rank_key(ld(row + c), c0 + c);
      if (key < last && key > best) best = key;
    }
    best = Red<G>::maxkey(best, red);
    if (lane == 0) emit(i, best);
    last = best;
  }
}

// ---- one thread per row: up to 64 classes ---------------------------------------------------------------------------------------
// A workgroup is one wave and takes 64 rows.  Rows side by side in memory (STAGED) come through LDS, so that the wave's loads
// are whole lines; classes that lie apart (maps) are loaded by the row's thread itself: neighbouring threads, neighbouring rows.
template <typename T> __device__ __forceinline__ void copy_to_lds(T* __restrict__ dst, const T* __restrict__ src, int n) {
  constexpr int E = 16 / sizeof(T);
  const int lane = threadIdx.x;
  int i = lane * E;
  for (; i + E <= n; i += 64 * E)
    *reinterpret_cast<Vec16*>(dst + i) = *reinterpret_cast<const LooseVec<T>*>(src + i);
  for (int e = n / E * E + lane; e < n; e += 64) dst[e] = src[e];
}
template <typename T> __device__ __forceinline__ void copy_from_lds(T* __restrict__ dst, const T* __restrict__ src, int n) {
  constexpr int E = 16 / sizeof(T);
  const int lane = threadIdx.x;
  for (int i = lane * E; i + E <= n; i += 64 * E)
    *reinterpret_cast<LooseVec<T>*>(dst + i) = *reinterpret_cast<const Vec16*>(src + i);
  for (int e = n / E * E + lane; e < n; e += 64) dst[e] = src[e];
}
// 64 rows that lie apart: one address for the wave and an offset of 32 bits for the lane (uh_apart checks that it fits), so that
// an access to a class takes a scalar addition and no registers.
struct ApartRows {
  long long base;             // elements, of the wave's first row
  uint32_t off;               // elements, the lane's row from there
  __device__ __forceinline__ ApartRows(const RowView& v, long long r0, int lane) {
    if (v.inner == 1) {
      base = r0 * v.so;
      off = (uint32_t)(lane * v.so);
      return;
    }
    const unsigned inner = (unsigned)v.inner;
    const unsigned o0 = __builtin_amdgcn_readfirstlane((unsigned)r0 / inner), i0 = (unsigned)r0 - o0 * inner;
    base = o0 * v.so + i0 * v.si;
    unsigned o = 0, i = i0 + lane;
    if (i0 + 63 >= inner) {
      o = i / inner;
      i -= o * inner;
    }
    off = (uint32_t)(o * v.so + ((long long)i - i0) * v.si);
  }
  template <typename T> __device__ __forceinline__ T* at(T* p, long long c_sc) const {
    return (T*)((char*)(p + base + c_sc) + (size_t)(off * (uint32_t)sizeof(T)));
  }
};
static inline bool uh_apart(const RowView& v, int elem) {
  const long long most = 0x7fffffffll / elem;
  if (v.inner == 1) return v.so < most / 64;
  if (v.si > most / 64 || v.inner > most / (v.si ? v.si : 1) || v.so > most) return false;
  return v.so >= (v.inner - 1) * v.si && (v.inner >= 64 ? v.so + 64 * v.si < most : v.so < most / 80);
}
// a row of C <= CREG classes to registers, -inf behind its end; p(c): where class c lies
template <typename T, int CREG, typename F>
__device__ __forceinline__ void load_classes(float (&x)[CREG], int C, F p) {
  C = renew_uniform(C);
#pragma unroll
  for (int c = 0; c < CREG; ++c) {
    x[c] = -INFINITY;
    if (c < C) x[c] = (float)*p(c);
  }
}
// the same from LDS; wide: rows start on 16 bytes and are at least that far apart
template <typename T, int CREG> __device__ __forceinline__ void load_classes_wide(float (&x)[CREG], const T* p, int C) {
  constexpr int E = 16 / sizeof(T);
#pragma unroll
  for (int c = 0; c < CREG; c += E)
    if (c < C) {
      alignas(16) T v[E];
      *reinterpret_cast<Vec16*>(v) = *reinterpret_cast<const Vec16*>(p + c);
#pragma unroll
      for (int j = 0; j < E; ++j) x[c + j] = c + j < C ? (float)v[j] : -INFINITY;
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) x[c + j] = -INFINITY;
    }
}
// FAR = false: the caller sums again what is_far
template <int CREG, bool ENT, bool FAR = true> __device__ __forceinline__ RowStat thread_row_stat(const float (&x)[CREG], int C, float c2) {
  C = renew_uniform(C);
  float m = x[0];
#pragma unroll
  for (int c = 1; c < CREG; c += 2)
    if (c < C) m = max3(m, x[c], c + 1 < CREG ? x[c + 1] : x[c]);
  if (m == -INFINITY) m = 0.f;
  float s = 0.f, t = 0.f;
  C = renew_uniform(C);
  const auto sums = [&](const auto& ref) {
#pragma unroll
    for (int c = 0; c < CREG; ++c)
      if (c < C) {
        const float z = ref.z(x[c]), e = ex2(z);
        s += e;
        if (ENT) {
          t = fmaf(e, fmaxf(z, UH_ZMIN), t);
          asm volatile("" : "+v"(s), "+v"(t));               // now: left to be summed later, the terms take two registers a class
        }
      }
  };
  if (FAR) with_ref(m, c2, sums);
  else sums(RowRef(m, c2));
  return RowStat{m, s, t};
}
// the same of a row of any length that one thread walks, 16 classes at a time, the next 16 on their way; each(x, c0) sees them
template <typename T, typename F>
__device__ __forceinline__ RowStat walk_row_stat(const T* __restrict__ p, long long sc, int C, float c2, F each) {
  constexpr int N = 16;
  RowStat a{0.f, 0.f, 0.f};
  T next[N];
  auto fetch = [&](int c0) {
#pragma unroll
    for (int j = 0; j < N; ++j) next[j] = c0 + j < C ? p[(c0 + j) * sc] : (T)-INFINITY;
  };
  fetch(0);
  for (int c0 = 0; c0 < C; c0 += N) {
    float x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = (float)next[j];
    if (c0 + N < C) fetch(c0 + N);
    a = join(a, thread_row_stat<N, true>(x, N, c2), c2);
    each(x, c0);
  }
  return a;
}

// ---- which kernel takes a call ---------------------------------------------------------------------------------------------
static inline int uh_elem_bytes(int dtype) { return dtype == UH_F32 ? 4 : 2; }
static inline unsigned uh_grid(long long blocks, long long most) { return (unsigned)(blocks < most ? blocks : most); }
// Logits that nothing reads soon again go past the caches: those of calls that no backward pass follows, and those that the card's
// last cache (256 MB) would not hold until it does (rows of 32000 bf16 classes with their gradient, through the caches and past
// them: 2000 rows 81 and 86 us, 4096 rows 174 and 172, 8192 rows 335 and 319; distillation 80 and 84, 176 and 176, 339 and 329).
static inline bool uh_read_once(const RowView& v, long long rows, int dtype, const float* stats) {
  return !stats || rows * v.C * uh_elem_bytes(dtype) > 1ll << 28;
}
enum { UH_GRID_WAVES = 256 * 32 };               // workgroups that loop over rows: 32 a CU

// Rows of at most 64 classes are a thread's: a group of 16 lanes, four loads each, would leave most lanes empty (12 classes of
// 16 bits: 2 of 16 at work).  10^6 rows of 12 bf16 classes by threads and by 16 lanes: log probabilities 11.5 and 87 us, a
// distillation loss of 3 slots 22 and 159 us; 300000 rows of 40: 10.6 and 27, 17.7 and 48 us.  STAGED needs one step from row to
// row, no more than 64 classes and a half further (LDS, and bytes read between the rows), and a dense gradient.  16 lanes take
// distillation's rows of 16 classes and more all the same
//   with eight slots and more, which the lanes share and a thread walks alone, three times over (166874 rows of 53 fp16 classes,
//   step, by threads and by 16 lanes: 8 slots 67 and 55 us, 22 slots 138 and 90 us; 24 fp32 classes, 8 slots: 42 and 44 us; 20
//   fp16 classes, 6 slots: 17 and 51 us);
//   where a thread's gradient, tile and table of the classes take more than 28 KB of LDS (300000 rows, 4 slots, step: fp32 32
//   classes 55 and 72 us, 48 classes 83 and 75, 64 classes 156 and 83; bf16 48 classes 50 and 82, 64 classes 90 and 82).
// Classes that lie apart are one address and a 32-bit offset a wave where that reaches (APART: 8 x 21 x 256 x 256 fp32, step: 27 us,
// walked: 75).  Elsewhere a thread walks its row from 4097 rows on; below, 256 lanes take a row, in lines of which they use an
// element (1000 fp32 classes, log probabilities, 256 lanes and one: 256 rows 5.3 and 59 us, 4096 rows 40 and 60, 16384 rows 158 and
// 60; 100 classes: 1024 rows 4.1 and 9.2, 4096 rows 8.5 and 9.0, 16384 rows 21 and 9.1).
enum ClassPath { PATH_GROUP, PATH_STAGED, PATH_APART, PATH_WALK, PATH_ANY };
static inline ClassPath uh_class_path(const RowView& v, const RowView* vo, long long rows, int dtype, int slots = 0) {
  const int elem = uh_elem_bytes(dtype);
  const bool side_by_side = v.sc == 1 && (!vo || vo->sc == 1);
  const bool shared = side_by_side && v.C >= 16 && (slots >= 8 || (slots && vo && v.C * 64 * (4 + 2 * elem) > 28672));
  if (v.C <= 64 && !shared) {
    const bool staged = v.sc == 1 && v.inner == 1 && v.so >= v.C && v.so <= 96 &&
                        (!vo || (vo->sc == 1 && vo->inner == 1 && vo->so == v.C));
    if (staged) return PATH_STAGED;
    if (uh_apart(v, elem) && (!vo || uh_apart(*vo, elem))) return PATH_APART;
    return rows > 4096 ? PATH_WALK : PATH_ANY;
  }
  if (side_by_side) return PATH_GROUP;
  return rows > 4096 ? PATH_WALK : PATH_ANY;
}

// A row is cut when it is longer than the `most` bytes that a workgroup of 256 is to hold in registers (at most 64 KB), or when
// there are too few rows to give every CU two workgroups; a part is then about 2048 classes (8 a lane) or more.  At most 64 parts: a
// wave joins them, one a lane.  bf16, up to 256 / 512 / 1024 workgroups: 32 x 32000 log probabilities 6.5 / 6.6 / 6.6 us, step of 16
// slots 11.5 / 12.0 / 12.0, 200 x 32000 log probabilities 10.7 / 10.6 / 9.2, step 19.7 / 19.1 / 18.6, 400 x 40000 16.7 / 16.9 / 14.4
// and 25.7 / 25.8 / 24.7 us (1024 are better for some hundreds of rows and cost 32 rows with alternatives nothing).  Parts of
// 1024 / 2048 / 4096 classes: 4 x 32000, top 20 17.1 / 14.6 / 14.0, loss 8.9 / 9.3 / 9.5, step 11.6 / 10.6 / 11.2 us.
// Parts are multiples of 64 classes, the last one what is left (at least one class; its loads may reach back into the part
// before it).
struct RowCut { int parts, len; };
static inline RowCut uh_cut_parts(int C, long long parts) {
  const int len = (int)(((C + parts - 1) / parts + 63) / 64 * 64);
  return RowCut{(C + len - 1) / len, len};
}
static inline RowCut uh_row_cut(long long rows, int C, int dtype, int most_bytes) {
  const int most = most_bytes / uh_elem_bytes(dtype);
  long long parts = (C + most - 1) / most;
  if (rows * parts < 512) {
    long long want = (512 + rows - 1) / rows;
    if (want > (C + 2047) / 2048) want = (C + 2047) / 2048;
    if (want > parts) parts = want;
  }
  if (parts > 64) parts = 64;
  return uh_cut_parts(C, parts);
}
