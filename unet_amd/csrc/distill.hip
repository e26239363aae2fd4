// Distillation from a teacher's top logits.  A row has a student's logits x over C classes and a teacher's slots
// (v_k, i_k), k < K: the logits (or log probabilities: a constant drops out) of a few of its best classes.  With
//     t = softmax over the slots of v / T,     p = softmax over the classes of x / T
//     loss_row = T^2 sum_k t_k (ln t_k - ln p[i_k]),          loss = scale * sum_rows w_row loss_row
//     dx_j = g scale w_row T (p_j - sum_{k: i_k = j} t_k)
// A slot with a negative index is free (t_k = 0).  Rows with w = 0 or without a filled slot count as 0 and get no
// gradient, whatever they hold.  A class index past C or a NaN among a row's slots makes that row's loss and gradient NaN.
//
// Sums over rows: every workgroup adds the rows it takes in 64 bits, one kernel adds the workgroups' sums, all in an order
// that the sizes alone decide.
#include "class_rows.h"
#include <stdlib.h>

struct DsArgs {
  RowView v, vo;
  long long rows;
  const void *value, *index;
  int K, value_dtype, index_bytes;
  const float* weight;
  float temperature, c2;
  // A row's loss without T^2 is a difference of logits over T, which may overflow where the loss itself does not (a class masked
  // with the type's lowest value, T < 1).  So it is taken in units of 1/unit, a power of two between T/32 and T/16, which costs
  // no bit: unit_t = unit / T, per_unit = 1 / unit.
  float unit, unit_t;
  double per_unit;
  float grad_scale;               // scale * grad_scale, or scale where gout is given
  const float* gout;
  float* stats;                   // [rows][2]: m, s
  bool once;                      // uh_read_once, for the loss alone (a step reads past the caches anyway)
  double* partial;

  __device__ __forceinline__ float weight_of(long long r) const { return weight ? weight[r] : 1.f; }
  __device__ __forceinline__ float value_of(long long e) const {
    return value_dtype == UH_F32    ? ((const float*)value)[e]
           : value_dtype == UH_BF16 ? (float)((const bf16*)value)[e]
                                    : (float)((const f16*)value)[e];
  }
  // slot k of a row: its class (-1: free, C: past the last one) and value (-inf where free, but a NaN stays one)
  __device__ __forceinline__ void slot(long long r, int k, float& val, int& cls) const {
    const long long e = v.entry(r, k, K);
    val = value_of(e);
    const long long i = load_int(index, index_bytes, e);
    cls = i < 0 ? -1 : i >= v.C ? v.C : (int)i;
    if (cls < 0 && val == val) val = -INFINITY;
  }
  // a row's loss of its sum_k t_k (ln t_k - ln p[i_k]) in units
  __device__ __forceinline__ double row_loss(float w, float kl) const { return (double)w * temperature * temperature * kl * per_unit; }
  __device__ __forceinline__ float coef(float w) const { return (gout ? gout[0] * grad_scale : grad_scale) * w * temperature; }
};

// t_k (ln t_k - ln p) of a slot, in units: vm is the teacher's maximum, sv the sum of its exponentials; the logarithms in units too
__device__ __forceinline__ float slot_term(float t, float val, float vm, float ln_sv, float x, float m, float ln_s, float unit_t) {
  return t > 0.f ? t * ((scaled(val, vm, unit_t) - ln_sv) - (scaled(x, m, unit_t) - ln_s)) : t == t ? 0.f : NAN;
}

// ---- a row by 16 lanes, or by any group with any strides: the slots in LDS -------------------------------------------------------
// The teacher's softmax of a row's slots into t_of / c_of [K].  Returns the sum of t (1, 0 without a filled slot, NaN).
struct Teacher { float vm, ln_sv, sum; };
template <int G> __device__ __forceinline__ Teacher group_teacher(const DsArgs& a, long long r, int lane, bool off, float* t_of, int* c_of,
                                                                  typename Red<G>::Buf& red) {
  float vm = -INFINITY, bad = 0.f;
  for (int k = lane; k < a.K; k += G) {
    float val = -INFINITY;
    int cls = -1;
    if (!off) a.slot(r, k, val, cls);
    t_of[k] = val, c_of[k] = cls;
    vm = fmaxf(vm, val);
    if (val != val || cls >= a.v.C) bad = 1.f;
  }
  vm = Red<G>::max_(vm, red);
  const float m = vm == -INFINITY ? 0.f : vm;
  float sv = 0.f, ln_sv;
  with_wave_ref(m, a.c2, [&](const auto& ref) {
    for (int k = lane; k < a.K; k += G) sv += ex2(ref.z(t_of[k]));
    Red<G>::sum2(sv, bad, red);
    const float inv = bad != 0.f ? NAN : sv == 0.f ? 0.f : rcp(sv);
    for (int k = lane; k < a.K; k += G) {
      const float val = t_of[k];
      t_of[k] = ex2(ref.z(val)) * inv;
    }
    ln_sv = ref.ln_s(m, sv) * a.unit;
  });
  return Teacher{m, ln_sv, bad != 0.f || !(sv >= 0.f) ? NAN : sv == 0.f ? 0.f : 1.f};
}
// sum_k t_k (ln t_k - ln p[i_k]), in units; the lanes read the slots' values again (t has taken their place)
template <typename T, int G> __device__ __forceinline__ float group_kl(const DsArgs& a, long long r, const T* __restrict__ row, int lane,
                                                                       const Teacher& q, const RowStat& s, const float* t_of, const int* c_of,
                                                                       typename Red<G>::Buf& red) {
  const float ln_s = s.s == 0.f ? 0.f : AnyRef(s.m, a.c2).ln_s(s.m, s.s) * a.unit;      // no class left: ln p = -inf
  float part = 0.f;
  if (!(q.sum == q.sum)) part = NAN;
  else if (q.sum != 0.f)
    for (int k = lane; k < a.K; k += G) {
      const float t = t_of[k];
      if (t != 0.f) part += slot_term(t, a.value_of(a.v.entry(r, k, a.K)), q.vm, q.ln_sv, ld(row + c_of[k] * a.v.sc), s.m, ln_s, a.unit_t);
    }
  return Red<G>::sum_(part, red);
}
// classes the teacher names, written again after the dense part: p minus what all slots of that class hold
template <typename T, int G, typename R> __device__ __forceinline__ void group_fix(const DsArgs& a, const T* __restrict__ row, T* __restrict__ out, int lane,
                                                                       float sum_t, float coef, const R& ref, float inv_s, const float* t_of,
                                                                       const int* c_of) {
  for (int k = lane; k < a.K; k += G) {
    const int c = c_of[k];
    if (c < 0 || c >= a.v.C) continue;
    float mine = 0.f;
    for (int j = 0; j < a.K; ++j) mine += c_of[j] == c ? t_of[j] : 0.f;
    st(out + c * a.vo.sc, coef * (sum_t * (ex2(ref.z(ld(row + c * a.v.sc))) * inv_s) - mine));
  }
}

// MODE 0: loss, 1: gradient with statistics given, 2: both.  Four rows of 16 lanes a wave: 100000 rows of 512 bf16 classes, 16
// slots, step: 69 us, by 64 lanes 127 (of 300, 8 slots, loss: 26 and 83 us).
template <typename T, int NV, int MODE>
__global__ __launch_bounds__(64) void ds_quad_kernel(DsArgs a, const T* __restrict__ x, T* __restrict__ dx) {
  extern __shared__ __align__(16) char lds[];
  Red<16>::Buf red;
  const int sub = threadIdx.x / 16, C = a.v.C;
  float* t_of = reinterpret_cast<float*>(lds) + sub * a.K;
  int* c_of = reinterpret_cast<int*>(lds) + (4 + sub) * a.K;
  const long long blocks = (a.rows + 3) / 4;
  double total = 0.0;
  for (long long b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int lane = renew(threadIdx.x % 16);
    const long long r = b * 4 + sub;
    const bool there = r < a.rows;
    const float w = there ? a.weight_of(r) : 0.f;
    const bool off = w == 0.f;
    const T* row = x + (there ? a.v.base(r) : 0);
    RowRegs<T, 16, NV> reg;
    if (!off) reg.load(row, 0, C, lane);
    const Teacher q = group_teacher<16>(a, r, lane, off, t_of, c_of, red);
    RowStat s{0.f, 0.f, 0.f};
    if constexpr (MODE == 1) {
      if (!off) s.m = a.stats[2 * r], s.s = a.stats[2 * r + 1];
    } else {
      s.m = group_max<16>(off ? -INFINITY : reg.lane_max(C));
      if (s.m == -INFINITY) s.m = 0.f;
      reg.fresh();
      with_wave_ref(s.m, a.c2, [&](const auto& ref) { reg.template lane_sums<false>(ref, C, s.s, s.t); });
      s.s = group_sum<16>(s.s);
      const float kl = group_kl<T, 16>(a, r, row, lane, q, s, t_of, c_of, red);
      if (lane == 0 && there) {
        if (!off && q.sum != 0.f) total += a.row_loss(w, kl);
        if (a.stats) { a.stats[2 * r] = off ? 0.f : s.m; a.stats[2 * r + 1] = off ? 0.f : s.s; }
      }
    }
    if constexpr (MODE != 0) {
      if (there) {
        T* out = dx + a.vo.base(r);
        const float inv_s = s.s == 0.f ? 0.f : rcp(s.s), co = a.coef(w), dense = co * q.sum * inv_s;
        reg.fresh();
        if (off || q.sum == 0.f) reg.map_store(out, 0, C, lane, [](float) { return 0.f; });
        else {
          with_wave_ref(s.m, a.c2, [&](const auto& ref) {
            reg.map_store(out, 0, C, lane, [&](float v) { return dense * ex2(ref.z(v)); });
            wave_stores_in_order();
            group_fix<T, 16>(a, row, out, lane, q.sum, co, ref, inv_s, t_of, c_of);
          });
        }
      }
    }
  }
  if constexpr (MODE != 1) {
    total += __shfl_xor(total, 16, 64);
    total += __shfl_xor(total, 32, 64);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = total;
  }
}

// ---- a row by one wave or by workgroups of 256: one wave holds the slots in its registers ------------------------------------------
// slot 64 q + lane of the row.  They are asked for before the row itself, so that their softmax is done while the row is on
// its way (a wave's loads come back in order).
struct SlotWave {
  float val[4], t[4], mine[4], xk[4];   // mine: what all slots of the same class hold; xk: the student's logit of the class
  int cls[4];
  float vm, ln_sv, sum;

  __device__ __forceinline__ void load(const DsArgs& a, long long r, int lane) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      val[q] = -INFINITY, cls[q] = -1;
      if (q * 64 < a.K && q * 64 + lane < a.K) a.slot(r, q * 64 + lane, val[q], cls[q]);
    }
  }
  __device__ __forceinline__ bool inside(const DsArgs& a, int q, int c0, int n) const {
    return cls[q] >= c0 && cls[q] < c0 + n && cls[q] < a.v.C;
  }
  // The slots' softmax, and the student's logits of their classes between c0 and c0 + n (in lines that the row's own loads,
  // issued before, bring).  t_of, c_of: K + 3 places, 16-byte aligned.
  template <typename T>
  __device__ __forceinline__ void softmax(const DsArgs& a, const T* __restrict__ row, int c0, int n, int lane, float* t_of, int* c_of,
                                          bool classes) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      xk[q] = 0.f;
      if (q * 64 < a.K && inside(a, q, c0, n)) xk[q] = ld(row + cls[q]);
    }
    float best = -INFINITY, sv = 0.f, bad = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q * 64 < a.K) {
        best = fmaxf(best, val[q]);
        if (val[q] != val[q] || cls[q] >= a.v.C) bad = 1.f;
      }
    best = group_max<64>(best);
    vm = best == -INFINITY ? 0.f : best;
    const AnyRef ref(vm, a.c2);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      t[q] = q * 64 < a.K ? ex2(ref.z(val[q])) : 0.f;
      sv += t[q];
    }
    sv = group_sum<64>(sv);
    const bool wrong = __any(bad != 0.f);
    const float inv = wrong ? NAN : sv == 0.f ? 0.f : rcp(sv);
#pragma unroll
    for (int q = 0; q < 4; ++q) t[q] *= inv;
    ln_sv = ref.ln_s(vm, sv) * a.unit;
    sum = wrong || !(sv >= 0.f) ? NAN : sv == 0.f ? 0.f : 1.f;
    if (!classes) return;
    const int K4 = (a.K + 3) / 4;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q * 64 < a.K && q * 64 + lane < 4 * K4) {
        t_of[q * 64 + lane] = t[q];
        c_of[q * 64 + lane] = cls[q];
      }
#pragma unroll
    for (int q = 0; q < 4; ++q) mine[q] = 0.f;
    __builtin_amdgcn_wave_barrier();
#pragma unroll 2
    for (int j = 0; j < K4; ++j) {
      const int4 c4 = reinterpret_cast<const int4*>(c_of)[j];
      const float4 t4 = reinterpret_cast<const float4*>(t_of)[j];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (q * 64 < a.K)
          mine[q] += ((c4.x == cls[q] ? t4.x : 0.f) + (c4.y == cls[q] ? t4.y : 0.f)) + ((c4.z == cls[q] ? t4.z : 0.f) + (c4.w == cls[q] ? t4.w : 0.f));
    }
  }
  // sum_k t_k (ln t_k - ln p[i_k]) in units, over the classes between c0 and c0 + n, in all lanes
  __device__ __forceinline__ float kl(const DsArgs& a, const RowStat& s, int c0, int n) const {
    const float ln_s = s.s == 0.f ? 0.f : AnyRef(s.m, a.c2).ln_s(s.m, s.s) * a.unit;    // no class left: ln p = -inf
    float part = 0.f;
    if (!(sum == sum)) part = NAN;
    else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (q * 64 < a.K && t[q] != 0.f && inside(a, q, c0, n)) part += slot_term(t[q], val[q], vm, ln_sv, xk[q], s.m, ln_s, a.unit_t);
    }
    return group_sum<64>(part);
  }
  // the classes the teacher names there, written again after the dense part
  template <typename T> __device__ __forceinline__ void fix(const DsArgs& a, T* __restrict__ out, int c0, int n, float coef, const AnyRef& ref,
                                                            float inv_s) const {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q * 64 < a.K && inside(a, q, c0, n)) st(out + cls[q], coef * (sum * (ex2(ref.z(xk[q])) * inv_s) - mine[q]));
  }
};
static inline size_t slot_lds(int K) { return (size_t)((K + 3) / 4 * 4) * 8; }

// one wave a row, up to 8 KB (bf16, by 64 and by 256 lanes: step 20000 x 2000, 16 slots 48 and 64 us, loss 10000 x 4096 25 and 30 us)
template <typename T, int NV, int MODE>
__global__ __launch_bounds__(64) void ds_wave_kernel(DsArgs a, const T* __restrict__ x, T* __restrict__ dx) {
  extern __shared__ __align__(16) char lds[];
  const int C = a.v.C, K4 = (a.K + 3) / 4 * 4;
  float* t_of = reinterpret_cast<float*>(lds);
  int* c_of = reinterpret_cast<int*>(lds) + K4;
  double total = 0.0;
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const int lane = renew(threadIdx.x);
    const float w = a.weight_of(r);
    RowRegs<T, 64, NV> reg;
    if (w == 0.f) {
      if (MODE != 0) reg.map_store(dx + a.vo.base(r), 0, C, lane, [](float) { return 0.f; });
      if (MODE != 1 && a.stats && lane == 0) { a.stats[2 * r] = 0.f; a.stats[2 * r + 1] = 0.f; }
      continue;
    }
    const T* row = x + a.v.base(r);
    SlotWave q;
    q.load(a, r, lane);
    reg.load(row, 0, C, lane);
    q.softmax(a, row, 0, C, lane, t_of, c_of, MODE != 0);
    RowStat s{0.f, 0.f, 0.f};
    if constexpr (MODE == 1) {
      s.m = a.stats[2 * r], s.s = a.stats[2 * r + 1];
    } else {
      s.m = group_max<64>(reg.lane_max(C));
      if (s.m == -INFINITY) s.m = 0.f;
      reg.fresh();
      with_ref(s.m, a.c2, [&](const auto& ref) { reg.template lane_sums<false>(ref, C, s.s, s.t); });
      s.s = group_sum<64>(s.s);
      const float kl = q.kl(a, s, 0, C);
      if (q.sum != 0.f) total += a.row_loss(w, kl);
      if (lane == 0 && a.stats) { a.stats[2 * r] = s.m; a.stats[2 * r + 1] = s.s; }
    }
    if constexpr (MODE != 0) {
      T* out = dx + a.vo.base(r);
      const float inv_s = s.s == 0.f ? 0.f : rcp(s.s), co = a.coef(w), dense = co * q.sum * inv_s;
      reg.fresh();
      if (q.sum == 0.f) reg.map_store(out, 0, C, lane, [](float) { return 0.f; });
      else {
        with_ref(s.m, a.c2, [&](const auto& ref) { reg.map_store(out, 0, C, lane, [&](float v) { return dense * ex2(ref.z(v)); }); });
        wave_stores_in_order();
        q.fix(a, out, 0, C, co, AnyRef(s.m, a.c2), inv_s);
      }
    }
  }
  if (MODE != 1 && threadIdx.x == 0) a.partial[blockIdx.x] = total;
}

// bf16, step: 4096 x 32000, 64 slots 117 us (525 MB, 4.5 TB/s), 2048 x 131072, 100 slots 277 us (1.07 GB, 3.9 TB/s); a copy that
// holds 16 vectors a thread reaches 5.1 TB/s: the loads stop while a row is joined and written.  fp16 1021 x 50021, 50 slots: loss
// 29 us, gradient 38 us.
// Long rows, or few: workgroups of 256 take a part of a row each.  The parts' (m, s) meet in memory, one 64-bit word a part
// that is written and read whole, so that no fence is needed: every workgroup that needs the row's statistics (all of them for
// a gradient, the first for the loss alone) waits for the other parts' words and keeps its own part in registers meanwhile: the
// row is read once.  A wait ends after `spins` looks at the latest: what is still missing then the waiting wave works out
// itself from the logits, operation for operation as the part's own workgroup does, so that no result depends on who did it and
// no workgroup on another one's being scheduled.
static constexpr unsigned long long UH_NO_WORD = ~0ull;          // m = s = a NaN that no arithmetic makes (0xffffffff)
__global__ __launch_bounds__(256) void ds_words_kernel(unsigned long long* __restrict__ words, long long n) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i < n) words[i] = UH_NO_WORD;
}
struct DsParts {
  int parts, len, spins;
  unsigned long long* words;
};

// Statistics of a part as 256 lanes make them (arriving_stat), by one wave, to the bit.  Kept small rather than fast: it stands
// where a part of a row waits in registers.
template <typename T> __device__ __forceinline__ RowStat alone_part_stat(const T* __restrict__ p, int c0, int n, float c2) {
  constexpr int E = 16 / sizeof(T);
  const int lane = threadIdx.x & 63;
  RowRegs<T, 256, 1> v;
  float m = -INFINITY;
#pragma unroll 1
  for (int at = 0; at < n * 4; at += 256 * E) {            // a quarter of the lanes a turn
    const int first = at / (1024 * E) * 256 * E, w = at / (256 * E) % 4;
    v.load(p, c0 + first, n - first, lane + 64 * w);
    m = fmaxf(m, v.lane_max(n - first));
  }
  m = group_max<64>(m);
  if (m == -INFINITY) m = 0.f;
  const bool far = is_far(m, c2);
  float total = 0.f;
#pragma unroll 1
  for (int w = 0; w < 4; ++w) {
    Online o;
#pragma unroll 1
    for (int first = 0; first < n; first += 256 * E) {
      v.load(p, c0 + first, n - first, lane + 64 * w);
      if (far) {
        float t0 = 0.f, t1 = 0.f;
        v.template add_sums<false>(FarRef(m, c2), n - first, o.s0, o.s1, t0, t1);
      } else {
        v.template online_vector<false>(0, c2, false, o);
      }
    }
    float s = o.s0 + o.s1;
    if (!far) s *= ex2(o.M - RowRef(m, c2).M);
    s = group_sum<64>(s);
    total = w == 0 ? s : total + s;
  }
  return RowStat{m, total == total ? total : NAN, 0.f};
}

template <typename T, int NV, int MODE>
__global__ __launch_bounds__(256) void ds_rows_kernel(DsArgs a, const T* __restrict__ x, T* __restrict__ dx, DsParts p) {
  extern __shared__ __align__(16) char lds[];
  __shared__ Red<256>::Buf red;
  __shared__ float joined[3];                              // m, s of the row; sum of t
  const int lane = threadIdx.x, wl = threadIdx.x & 63, K4 = (a.K + 3) / 4 * 4;
  float* t_of = reinterpret_cast<float*>(lds);
  int* c_of = reinterpret_cast<int*>(lds) + K4;
  const long long r = blockIdx.y + (long long)blockIdx.z * 32768;
  if (r >= a.rows) return;
  const int part = blockIdx.x, c0 = part * p.len, n = min(p.len, a.v.C - c0);
  const bool first = serial_wave<256>();                   // the wave with the slots
  const float w = a.weight_of(r);
  T* out = MODE != 0 ? dx + a.vo.base(r) : nullptr;
  RowRegs<T, 256, NV> reg;
  if (w == 0.f) {
    if (MODE != 0) reg.map_store(out, c0, n, lane, [](float) { return 0.f; });
    if (MODE != 1 && lane == 0) {
      if (MODE == 2 || part == 0) a.partial[MODE == 2 ? r * p.parts + part : r] = 0.0;
      if (MODE == 0 && part == 0 && a.stats) { a.stats[2 * r] = 0.f; a.stats[2 * r + 1] = 0.f; }
    }
    return;
  }
  const T* row = x + a.v.base(r);
  SlotWave q;
  const bool slots = first && (MODE != 0 || part == 0);
  if (slots) q.load(a, r, wl);
  if (MODE == 2 || (MODE == 0 && a.once)) reg.template load<true>(row, c0, n, lane);
  else reg.load(row, c0, n, lane);
  if (slots) {
    // the loss alone is the first part's to work out; for a gradient every part has its classes' share of it
    if (MODE == 0) q.softmax(a, row, 0, a.v.C, wl, t_of, c_of, false);
    else q.softmax(a, row, c0, n, wl, t_of, c_of, true);
    if (wl == 0) joined[2] = q.sum;
  }
  RowStat s{0.f, 0.f, 0.f};
  if constexpr (MODE == 1) {
    s.m = a.stats[2 * r], s.s = a.stats[2 * r + 1];
    __syncthreads();                                       // joined[2]
  } else {
    float lane_top;
    s = arriving_stat<T, 256, NV, false, 0>(reg, a.c2, n, lane_top, nullptr, red);
    if (s.s != s.s) s.s = NAN;                             // never the bits of UH_NO_WORD
    if (p.parts > 1) {
      unsigned long long* words = p.words + r * p.parts;
      if (lane == 0)
        __hip_atomic_store(words + part, (unsigned long long)__float_as_uint(s.s) << 32 | __float_as_uint(s.m), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
      if (MODE == 0 && part != 0) return;
      if (first) {
        unsigned long long word = wl == part ? (unsigned long long)__float_as_uint(s.s) << 32 | __float_as_uint(s.m) : UH_NO_WORD;
        const bool other = wl < p.parts && wl != part;
        for (int i = 0; i < p.spins; ++i) {
          if (other && word == UH_NO_WORD) word = __hip_atomic_load(words + wl, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          if (!__any(other && word == UH_NO_WORD)) break;
          __builtin_amdgcn_s_sleep(2);
        }
        for (unsigned long long left = __ballot(other && word == UH_NO_WORD); left; left &= left - 1) {
          const int who = __ffsll(left) - 1, at = who * p.len;
          const RowStat u = alone_part_stat<T>(row, at, min(p.len, a.v.C - at), a.c2);
          if (wl == who) word = (unsigned long long)__float_as_uint(u.s) << 32 | __float_as_uint(u.m);
        }
        RowStat j{__uint_as_float((uint32_t)word), wl < p.parts ? __uint_as_float((uint32_t)(word >> 32)) : 0.f, 0.f};
        if (wl >= p.parts) j.m = 0.f;
        for (int o = 1; o < 64 && o < p.parts; o <<= 1) {
          const RowStat u{__shfl_xor(j.m, o, 64), __shfl_xor(j.s, o, 64), 0.f};
          j = wl & o ? join(u, j, a.c2) : join(j, u, a.c2);
        }
        if (wl == 0) joined[0] = j.m, joined[1] = j.s;
      }
      __syncthreads();
      s.m = joined[0], s.s = joined[1];
    }
  }
  const float sum_t = joined[2];
  if constexpr (MODE != 0) {
    const float inv_s = s.s == 0.f ? 0.f : rcp(s.s), co = a.coef(w), dense = co * sum_t * inv_s;
    if (sum_t == 0.f) reg.map_store(out, c0, n, lane, [](float) { return 0.f; });
    else {
      with_ref(s.m, a.c2, [&](const auto& ref) { reg.map_store(out, c0, n, lane, [&](float v) { return dense * ex2(ref.z(v)); }); });
      __syncthreads();                                     // another wave may have written the class
      if (first) q.fix(a, out, c0, n, co, AnyRef(s.m, a.c2), inv_s);
    }
  }
  if (MODE != 1 && first) {
    const float kl = MODE == 0 ? q.kl(a, s, 0, a.v.C) : q.kl(a, s, c0, n);
    if (wl == 0) {
      a.partial[MODE == 2 ? r * p.parts + part : r] = sum_t != 0.f ? a.row_loss(w, kl) : 0.0;
      if (MODE == 0 && a.stats) { a.stats[2 * r] = s.m; a.stats[2 * r + 1] = s.s; }
    }
  }
}

// ---- one thread per row ----------------------------------------------------------------------------------------------------------
// The teacher's softmax of a thread's own row.  KS > 0: at most KS slots, read once and kept; KS = 0: any number, read once for
// the maximum, once for the sum and again for every use.  Kept in 4 places and read again, step, 8 x 21 x 256 x 256 fp32: 1 slot 29.3
// and 31.3 us, 2 32.3 and 35.1, 4 36.2 and 42.8; 2^20 x 12 bf16: 4 slots 38.9 and 54.1.  Kept in 8 places (no such instance) and
// read again: 5 slots 38.9 and 46.4 us, 8 slots 44.8 and 44.9.
// R: RowRef, where the caller sees to the rows for which it will not do, or AnyRef.
template <int KS, typename R> struct ThreadTeacher {
  float vm, ln_sv, inv, sum;
  R ref;
  float val_[KS > 0 ? KS : 1];
  int cls_[KS > 0 ? KS : 1];
  template <typename F> __device__ __forceinline__ void each(const DsArgs& a, long long r, F f) const {
    if constexpr (KS > 0) {
#pragma unroll
      for (int k = 0; k < KS; ++k)
        if (k < a.K) f(val_[k], cls_[k]);
    } else {
      for (int k = 0; k < a.K; ++k) {
        float val;
        int cls;
        a.slot(r, k, val, cls);
        f(val, cls);
      }
    }
  }
  __device__ __forceinline__ ThreadTeacher(const DsArgs& a) : ref(0.f, a.c2) {}
  // asks for the slots; what comes of them follows in softmax
  __device__ __forceinline__ void fetch(const DsArgs& a, long long r) {
    if constexpr (KS > 0) {
#pragma unroll
      for (int k = 0; k < KS; ++k)
        if (k < a.K) a.slot(r, k, val_[k], cls_[k]);
    }
  }
  __device__ __forceinline__ void softmax(const DsArgs& a, long long r, float w) {
    float best = -INFINITY, sv = 0.f;
    bool bad = false;
    if (w != 0.f) {
      each(a, r, [&](float val, int cls) {
        bad |= val != val || cls >= a.v.C;
        best = fmaxf(best, val);
      });
      if (best == -INFINITY) best = 0.f;
      ref = R(best, a.c2);
      each(a, r, [&](float val, int) { sv += ex2(ref.z(val)); });
    }
    vm = best;
    inv = bad ? NAN : sv == 0.f ? 0.f : rcp(sv);
    ln_sv = w != 0.f ? ref.ln_s(vm, sv) * a.unit : 0.f;
    sum = bad || !(sv >= 0.f) ? NAN : sv == 0.f ? 0.f : 1.f;
  }
  __device__ __forceinline__ float t(float val) const { return ex2(ref.z(val)) * inv; }
};
// at(c): where the student's class c lies
template <int KS, typename R, typename F>
__device__ __forceinline__ float thread_kl(const DsArgs& a, long long r, const ThreadTeacher<KS, R>& q, const RowStat& s, F at) {
  if (!(q.sum == q.sum)) return NAN;
  const float ln_s = s.s == 0.f ? 0.f : R(s.m, a.c2).ln_s(s.m, s.s) * a.unit;  // no class left: ln p = -inf
  float kl = 0.f;
  q.each(a, r, [&](float val, int cls) {
    const float t = q.t(val);
    // (a free slot has t = 0: its exponent is -inf, or a NaN where a RowRef's M is -inf, and then the sum is one as well)
    if (t != 0.f) kl += slot_term(t, val, q.vm, q.ln_sv, ld(at(cls)), s.m, ln_s, a.unit_t);
  });
  return kl;
}
__device__ __forceinline__ double wave_total(double v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// MODE 0: loss, 1: gradient with statistics given, 2: both.  Up to 64 classes.  A thread's row lies in LDS as well (tab, [C][64]:
// no bank is asked twice): first the logits, out of which the slots pick theirs (from memory, apart, 64 classes are 64 lines),
// then what the teacher holds of each class, so that a class named twice costs nothing and every gradient is rounded once.
// 32 x 21 x 256 x 256 fp32, 4 slots, step: 97 us (419 MB, 4.3 TB/s); 2^20 rows of 12 bf16 classes, 3 slots, loss: 22 us (50 MB),
// bound by its arithmetic and by what each slot looks up, not by memory.
template <typename T, int CREG, bool STAGED, int MODE, int KS>
__global__ __launch_bounds__(64) void ds_thread_kernel(DsArgs a, const T* __restrict__ x, T* __restrict__ dx, bool wide) {
  extern __shared__ __align__(16) char lds[];
  constexpr int E = 16 / sizeof(T);
  const int lane = threadIdx.x, C = a.v.C, so = (int)a.v.so;
  float* tab = reinterpret_cast<float*>(lds);                                     // [C][64]
  T* tile = reinterpret_cast<T*>(lds + (MODE != 0 || !STAGED ? (size_t)C * 64 * 4 : 0));
  T* res = tile + (64 * so + E - 1) / E * E;                                       // STAGED, MODE > 0: the gradient on its way out
  const long long blocks = (a.rows + 63) / 64;
  double total = 0.0;
  for (long long b = blockIdx.x; b < blocks; b += gridDim.x) {
    const long long r = b * 64 + lane;
    const int here = (int)min(64ll, a.rows - b * 64);
    ThreadTeacher<KS, RowRef> q(a);
    float w = 0.f;
    if (lane < here) {
      w = a.weight_of(r);
      q.fetch(a, r);
    }
    if constexpr (STAGED) {
      __syncthreads();
      copy_to_lds(tile, x + b * 64 * so, (here - 1) * so + C);
      __syncthreads();
    }
    const ApartRows from(a.v, b * 64, lane);
    const auto at = [&](int c) { return STAGED ? tile + lane * so + c : from.at(x, c * a.v.sc); };
    if (lane < here) {
      float v[CREG];
      if (STAGED && wide) load_classes_wide<T, CREG>(v, tile + lane * so, C);
      else load_classes<T, CREG>(v, C, at);
      q.softmax(a, r, w);
      // a far maximum (class_rows.h) in either row: what the sweeps below make of it is worked out again, class by class and
      // slot by slot, so that other rows pay a comparison
      bool far = is_far(q.vm, a.c2);
      const bool on = w != 0.f && (q.sum != 0.f || far);
      RowStat s{0.f, 0.f, 0.f};
      if (on) {
        if (MODE == 1) s.m = a.stats[2 * r], s.s = a.stats[2 * r + 1];
        else s = thread_row_stat<CREG, false, false>(v, C, a.c2);
        far |= is_far(s.m, a.c2);
      }
      if (MODE != 1) {
        if (on) {
          float kl;
          if constexpr (STAGED) kl = thread_kl(a, r, q, s, [&](int c) { return tile + lane * so + c; });
          else {
            const int n = renew_uniform(C);
#pragma unroll
            for (int c = 0; c < CREG; ++c)
              if (c < n) tab[c * 64 + lane] = v[c];
            kl = thread_kl(a, r, q, s, [&](int c) { return tab + c * 64 + lane; });
          }
          if (__builtin_expect(far, 0)) {
            const AnyRef ref(s.m, a.c2);
            s.s = 0.f;
            for (int c = 0; c < C; ++c) s.s += ex2(ref.z(ld(at(c))));
            ThreadTeacher<0, AnyRef> f(a);
            f.softmax(a, r, w);
            kl = thread_kl(a, r, f, s, at);
          }
          total += a.row_loss(w, kl);
        }
        if (a.stats) { a.stats[2 * r] = s.m; a.stats[2 * r + 1] = s.s; }
      }
      if constexpr (MODE != 0) {
        const ApartRows to_rows(a.vo, b * 64, lane);
        const auto to = [&](int c) { return STAGED ? res + lane * C + c : to_rows.at(dx, c * a.vo.sc); };
        if (!on) {
          for (int c = 0; c < C; ++c) *to(c) = (T)0.f;
        } else {
          const RowRef ref(s.m, a.c2);
          const float inv_s = s.s == 0.f ? 0.f : rcp(s.s), co = a.coef(w), dense = co * q.sum * inv_s;
          const auto named = [&](const auto& teacher) {
#pragma unroll 8
            for (int c = 0; c < C; ++c) tab[c * 64 + lane] = 0.f;
            teacher.each(a, r, [&](float val, int cls) {
              if (cls >= 0 && cls < C) tab[cls * 64 + lane] -= teacher.t(val);
            });
          };
          named(q);
          const int n = renew_uniform(C);
#pragma unroll
          for (int c = 0; c < CREG; ++c)
            if (c < n) *to(c) = (T)fmaf(co, tab[c * 64 + lane], dense * ex2(ref.z(v[c])));
          if (__builtin_expect(far, 0)) {
            const AnyRef any(s.m, a.c2);
            ThreadTeacher<0, AnyRef> f(a);
            f.softmax(a, r, w);
            named(f);
            for (int c = 0; c < C; ++c) *to(c) = (T)fmaf(co, tab[c * 64 + lane], co * f.sum * inv_s * ex2(any.z(ld(at(c)))));
          }
        }
      }
    }
    if (STAGED && MODE != 0) {
      __syncthreads();
      copy_from_lds(dx + b * 64 * C, res, here * C);
    }
  }
  if (MODE != 1) {
    total = wave_total(total);
    if (lane == 0) a.partial[blockIdx.x] = total;
  }
}

// more classes, lying apart: the thread walks its row
template <typename T, int MODE> __global__ __launch_bounds__(64) void ds_walk_kernel(DsArgs a, const T* __restrict__ x, T* __restrict__ dx) {
  const int C = a.v.C;
  const long long sc = a.v.sc, osc = a.vo.sc, blocks = (a.rows + 63) / 64;
  double total = 0.0;
  for (long long b = blockIdx.x; b < blocks; b += gridDim.x) {
    const long long r = b * 64 + threadIdx.x;
    if (r >= a.rows) continue;
    const T* row = x + a.v.base(r);
    const float w = a.weight_of(r);
    ThreadTeacher<0, AnyRef> q(a);
    q.softmax(a, r, w);
    const bool on = w != 0.f && q.sum != 0.f;
    RowStat s{0.f, 0.f, 0.f};
    if (on) {
      if (MODE == 1) s.m = a.stats[2 * r], s.s = a.stats[2 * r + 1];
      else s = walk_row_stat(row, sc, C, a.c2, [](const float (&)[16], int) {});
    }
    if (MODE != 1) {
      if (on) total += a.row_loss(w, thread_kl(a, r, q, s, [&](int c) { return row + c * sc; }));
      if (a.stats) { a.stats[2 * r] = s.m; a.stats[2 * r + 1] = s.s; }
    }
    if constexpr (MODE != 0) {
      T* out = dx + a.vo.base(r);
      const AnyRef ref(s.m, a.c2);
      const float inv_s = s.s == 0.f ? 0.f : rcp(s.s), co = a.coef(w), dense = co * q.sum * inv_s;
      constexpr int N = 16;
      T next[N];
      auto fetch = [&](int c0) {
#pragma unroll
        for (int j = 0; j < N; ++j) next[j] = c0 + j < C && on ? row[(c0 + j) * sc] : (T)0.f;
      };
      fetch(0);
      for (int c0 = 0; c0 < C; c0 += N) {
        float v[N];
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = (float)next[j];
        if (c0 + N < C) fetch(c0 + N);
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (c0 + j < C) st(out + (c0 + j) * osc, on ? dense * ex2(ref.z(v[j])) : 0.f);
      }
      if (on)
        for (int k = 0; k < a.K; ++k) {
          float val, mine = 0.f;
          int cls;
          a.slot(r, k, val, cls);
          if (cls < 0 || cls >= C) continue;
          q.each(a, r, [&](float v, int other) { mine += other == cls ? q.t(v) : 0.f; });
          st(out + cls * osc, co * (q.sum * (ex2(ref.z(ld(row + cls * sc))) * inv_s) - mine));
        }
    }
  }
  if (MODE != 1) {
    total = wave_total(total);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = total;
  }
}

// ---- one workgroup per row, any strides ----------------------------------------------------------------------------------------
template <typename T, int MODE> __global__ __launch_bounds__(256) void ds_any_kernel(DsArgs a, const T* __restrict__ x, T* __restrict__ dx) {
  extern __shared__ __align__(16) char lds[];
  float* t_of = reinterpret_cast<float*>(lds);
  int* c_of = reinterpret_cast<int*>(lds) + a.K;
  __shared__ Red<256>::Buf red;
  const int lane = threadIdx.x, C = a.v.C;
  double total = 0.0;
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const float w = a.weight_of(r);
    const T* row = x + a.v.base(r);
    __syncthreads();
    const Teacher q = group_teacher<256>(a, r, lane, w == 0.f, t_of, c_of, red);
    const bool on = q.sum != 0.f;
    RowStat s{0.f, 0.f, 0.f};
    if (on) {
      if (MODE == 1) s.m = a.stats[2 * r], s.s = a.stats[2 * r + 1];
      else s = strided_row_stat<T, 256>(row, C, a.v.sc, a.c2, lane, red);
    }
    if (MODE != 1) {
      const float kl = group_kl<T, 256>(a, r, row, lane, q, s, t_of, c_of, red);
      if (lane == 0) {
        if (on) total += a.row_loss(w, kl);
        if (a.stats) { a.stats[2 * r] = s.m; a.stats[2 * r + 1] = s.s; }
      }
    }
    if constexpr (MODE != 0) {
      T* out = dx + a.vo.base(r);
      const AnyRef ref(s.m, a.c2);
      const float inv_s = s.s == 0.f ? 0.f : rcp(s.s), co = a.coef(w), dense = co * q.sum * inv_s;
      for (int c = lane; c < C; c += 256) st(out + c * a.vo.sc, on ? dense * ex2(ref.z(ld(row + c * a.v.sc))) : 0.f);
      __syncthreads();
      if (on) group_fix<T, 256>(a, row, out, lane, q.sum, co, ref, inv_s, t_of, c_of);
    }
  }
  if (MODE != 1 && lane == 0) a.partial[blockIdx.x] = total;
}

__global__ __launch_bounds__(1024) void ds_finish_kernel(long long n, const double* __restrict__ partial, double scale, float* __restrict__ loss) {
  __shared__ double buf[16];
  double v = 0.0;
  for (long long i = threadIdx.x; i < n; i += 1024) v += partial[i];
  v = wave_total(v);
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) v += buf[w];
    loss[0] = (float)(v * scale);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------
static int distill_check(const char* who, const uh_class_view* v, const void* logits, const uh_slots* sl, float temperature) {
  const int ok = uh_check_view(v, who);
  if (ok != UH_OK) return ok;
  UH_REQUIRE(sl, "%s: no slots", who);
  UH_REQUIRE(sl->slots > 0 && sl->slots <= UH_SLOTS_MAX, "%s: %d slots (1 to %d)", who, sl->slots, UH_SLOTS_MAX);
  UH_REQUIRE(sl->value_dtype >= UH_F32 && sl->value_dtype <= UH_F16, "%s: slot dtype %d", who, sl->value_dtype);
  UH_REQUIRE(sl->index_bytes == 4 || sl->index_bytes == 8, "%s: slot indices of %d bytes", who, sl->index_bytes);
  UH_REQUIRE(logits && sl->value && sl->index, "%s: null pointer", who);
  UH_REQUIRE(uh_temperature(temperature), "%s: temperature %g (1e-6 to 1e6)", who, temperature);
  return UH_OK;
}

static int same_rows(const char* who, const uh_class_view* v, const uh_class_view* o) {
  const int ok = uh_check_view(o, who);
  if (ok != UH_OK) return ok;
  UH_REQUIRE(o->dtype == v->dtype && o->classes == v->classes && o->outer == v->outer && o->inner == v->inner,
             "%s: the gradient's view differs from the logits'", who);
  return UH_OK;
}

static DsArgs ds_args(const uh_class_view* view, const uh_class_view* out, const uh_slots* s, const float* weight, float temperature) {
  DsArgs a;
  a.v = uh_row_view(view), a.vo = uh_row_view(out);
  a.rows = view->outer * view->inner;
  a.value = s->value, a.index = s->index, a.K = s->slots, a.value_dtype = s->value_dtype, a.index_bytes = s->index_bytes;
  int e;
  frexpf(temperature, &e);                                 // 2^(e-1) <= T < 2^e
  a.unit = ldexpf(1.f, e - 5), a.unit_t = 1.f / temperature * a.unit, a.per_unit = ldexp(1.0, 5 - e);
  a.weight = weight, a.temperature = temperature, a.c2 = (float)(1.4426950408889634 / (double)temperature);
  a.grad_scale = 0.f, a.gout = nullptr, a.stats = nullptr, a.partial = nullptr, a.once = false;
  return a;
}

// How a call's rows are taken, and its workspace: partial sums (one a workgroup), then the words of rows in parts.
struct DsPlan {
  ClassPath path;
  RowCut cut;
  bool parts;                     // rows by workgroups of 256
  size_t words_at, bytes;
};
static DsPlan ds_plan(const RowView& v, const RowView* vo, long long rows, int dtype, int slots, bool step) {
  DsPlan p;
  const int elem = uh_elem_bytes(dtype);
  p.path = uh_class_path(v, vo, rows, dtype, slots);
  p.parts = p.path == PATH_GROUP && (long long)v.C * elem > 8192;
  p.cut = p.parts ? uh_row_cut(rows, v.C, dtype, step ? 65536 : 32768) : RowCut{1, v.C};
  const size_t sums = p.parts && rows * p.cut.parts > UH_GRID_WAVES ? rows * p.cut.parts : UH_GRID_WAVES;
  p.words_at = (sums * sizeof(double) + 15) / 16 * 16;
  p.bytes = p.words_at + (p.cut.parts > 1 ? (size_t)rows * p.cut.parts * 8 : 0);
  return p;
}

static int ds_spins() {
  const char* e = getenv("UNET_AMD_DISTILL_SPINS");
  return e ? atoi(e) : 1 << 14;
}

// MODE 0: loss, 1: gradient, 2: both; returns how many partial sums there are
template <typename T, int MODE> static long long ds_launch(const DsArgs& a, const T* x, T* dx, const DsPlan& p, char* ws, hipStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const int C = a.v.C;
  const long long rows = a.rows;
  const unsigned waves = uh_grid((rows + 63) / 64, UH_GRID_WAVES), blocks = uh_grid(rows, UH_GRID_WAVES);
  if (p.path == PATH_STAGED || p.path == PATH_APART) {
    const bool staged = p.path == PATH_STAGED, wide = staged && (a.v.so * sizeof(T)) % 16 == 0;
    const size_t lds = (MODE != 0 || !staged ? (size_t)C * 64 * 4 : 0) + (staged ? ((64 * a.v.so + E - 1) / E * E + (MODE ? 64 * C : 0)) * sizeof(T) : 0);
#define UH_GO3(R, ST, KS) hipLaunchKernelGGL((ds_thread_kernel<T, R, ST, MODE, KS>), dim3(waves), dim3(64), lds, s, a, x, dx, wide)
#define UH_GO2(R, ST) do { if (a.K <= 4) UH_GO3(R, ST, 4); else UH_GO3(R, ST, 0); } while (0)
#define UH_GO(ST) do { if (C <= 16) UH_GO2(16, ST); else if (C <= 32) UH_GO2(32, ST); else UH_GO2(64, ST); } while (0)
    if (staged) UH_GO(true); else UH_GO(false);
#undef UH_GO
#undef UH_GO2
#undef UH_GO3
    return (int)waves;
  }
  if (p.path == PATH_WALK) {
    hipLaunchKernelGGL((ds_walk_kernel<T, MODE>), dim3(waves), dim3(64), 0, s, a, x, dx);
    return (int)waves;
  }
  if (p.path == PATH_ANY) {
    hipLaunchKernelGGL((ds_any_kernel<T, MODE>), dim3(blocks), dim3(256), (size_t)a.K * 8, s, a, x, dx);
    return (int)blocks;
  }
  if (C <= 16 * 4 * E) {
    const unsigned quads = uh_grid((rows + 3) / 4, UH_GRID_WAVES);
    hipLaunchKernelGGL((ds_quad_kernel<T, 4, MODE>), dim3(quads), dim3(64), (size_t)a.K * 32, s, a, x, dx);
    return (int)quads;
  }
  if (!p.parts) {
    if (C <= 64 * 4 * E) hipLaunchKernelGGL((ds_wave_kernel<T, 4, MODE>), dim3(blocks), dim3(64), slot_lds(a.K), s, a, x, dx);
    else hipLaunchKernelGGL((ds_wave_kernel<T, 8, MODE>), dim3(blocks), dim3(64), slot_lds(a.K), s, a, x, dx);
    return (int)blocks;
  }
  // a gradient alone needs no joining: its parts are as long as suits a copy
  const RowCut cut = MODE == 1 ? uh_cut_parts(C, (C + 256 * 4 * E - 1) / (256 * 4 * E)) : p.cut;
  DsParts q{cut.parts, cut.len, 0, nullptr};
  if (MODE != 1 && cut.parts > 1) {
    q.spins = ds_spins();
    q.words = (unsigned long long*)(ws + p.words_at);
    const long long n = rows * cut.parts;
    hipLaunchKernelGGL(ds_words_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, q.words, n);
  }
  const dim3 grid((unsigned)cut.parts, (unsigned)(rows < 32768 ? rows : 32768), (unsigned)((rows + 32767) / 32768));
#define UH_GO(NV) hipLaunchKernelGGL((ds_rows_kernel<T, NV, MODE>), grid, dim3(256), slot_lds(a.K), s, a, x, dx, q)
  // parts of 32 bits are longer than 1024 classes; those of the loss alone longer than 32 KB only where 64 of 32 KB are not
  // enough (more than 524288 classes of 32 bits)
  if constexpr (MODE == 1) UH_GO(4);
  else if (cut.len <= 256 * 4 * E) {
    if constexpr (sizeof(T) == 2) { if (cut.len <= 256 * E) UH_GO(1); else UH_GO(4); }
    else UH_GO(4);
  } else if (cut.len <= 256 * 8 * E) UH_GO(8);
  else if constexpr (MODE == 2 || sizeof(T) == 4) UH_GO(16);
#undef UH_GO
  return MODE == 2 ? (long long)rows * cut.parts : rows;
}

template <int MODE> static long long ds_dispatch(const DsArgs& a, int dtype, const void* x, void* dx, const DsPlan& p, void* ws, hipStream_t s) {
  if (dtype == UH_F32) return ds_launch<float, MODE>(a, (const float*)x, (float*)dx, p, (char*)ws, s);
  if (dtype == UH_BF16) return ds_launch<bf16, MODE>(a, (const bf16*)x, (bf16*)dx, p, (char*)ws, s);
  return ds_launch<f16, MODE>(a, (const f16*)x, (f16*)dx, p, (char*)ws, s);
}

extern "C" size_t uh_topk_distill_workspace(const uh_class_view* view) {
  if (uh_check_view(view, "topk_distill_workspace") != UH_OK) return 0;
  const RowView v = uh_row_view(view);
  const size_t loss = ds_plan(v, nullptr, view->outer * view->inner, view->dtype, 0, false).bytes;
  const size_t step = ds_plan(v, nullptr, view->outer * view->inner, view->dtype, 0, true).bytes;
  return loss > step ? loss : step;
}

extern "C" int uh_topk_distill(const uh_class_view* view, const void* logits, const uh_slots* slots, const float* weight,
                               float temperature, double scale, float* loss, float* stats, void* workspace,
                               size_t workspace_bytes, uh_stream s) {
  const int ok = distill_check("topk_distill", view, logits, slots, temperature);
  if (ok != UH_OK) return ok;
  UH_REQUIRE(loss && workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= uh_topk_distill_workspace(view),
             "topk_distill: null pointer or workspace of %zu bytes", workspace_bytes);
  DsArgs a = ds_args(view, view, slots, weight, temperature);
  a.stats = stats, a.partial = (double*)workspace;
  a.once = uh_read_once(a.v, a.rows, view->dtype, stats);
  const DsPlan p = ds_plan(a.v, nullptr, a.rows, view->dtype, a.K, false);
  const long long n = ds_dispatch<0>(a, view->dtype, logits, nullptr, p, workspace, (hipStream_t)s);
  hipLaunchKernelGGL(ds_finish_kernel, dim3(1), dim3(1024), 0, (hipStream_t)s, n, (const double*)workspace, scale, loss);
  return uh_check_launch("topk_distill");
}

extern "C" int uh_topk_distill_bwd(const uh_class_view* view, const uh_class_view* out_view, const void* logits,
                                   const uh_slots* slots, const float* weight, float temperature, double scale,
                                   const float* gout, const float* stats, void* dlogits, uh_stream s) {
  int ok = distill_check("topk_distill_bwd", view, logits, slots, temperature);
  if (ok == UH_OK) ok = same_rows("topk_distill_bwd", view, out_view);
  if (ok != UH_OK) return ok;
  UH_REQUIRE(gout && stats && dlogits, "topk_distill_bwd: null pointer");
  DsArgs a = ds_args(view, out_view, slots, weight, temperature);
  a.gout = gout, a.grad_scale = (float)scale, a.stats = const_cast<float*>(stats);
  const DsPlan p = ds_plan(a.v, &a.vo, a.rows, view->dtype, a.K, false);
  ds_dispatch<1>(a, view->dtype, logits, dlogits, p, nullptr, (hipStream_t)s);
  return uh_check_launch("topk_distill_bwd");
}

extern "C" int uh_topk_distill_step(const uh_class_view* view, const uh_class_view* out_view, const void* logits,
                                    const uh_slots* slots, const float* weight, float temperature, double scale,
                                    float grad_scale, float* loss, void* dlogits, void* workspace, size_t workspace_bytes,
                                    uh_stream s) {
  int ok = distill_check("topk_distill_step", view, logits, slots, temperature);
  if (ok == UH_OK) ok = same_rows("topk_distill_step", view, out_view);
  if (ok != UH_OK) return ok;
  UH_REQUIRE(loss && dlogits && workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= uh_topk_distill_workspace(view),
             "topk_distill_step: null pointer or workspace of %zu bytes", workspace_bytes);
  DsArgs a = ds_args(view, out_view, slots, weight, temperature);
  a.grad_scale = (float)(scale * (double)grad_scale), a.partial = (double*)workspace;
  const DsPlan p = ds_plan(a.v, &a.vo, a.rows, view->dtype, a.K, true);
  const long long n = ds_dispatch<2>(a, view->dtype, logits, dlogits, p, workspace, (hipStream_t)s);
  hipLaunchKernelGGL(ds_finish_kernel, dim3(1), dim3(1024), 0, (hipStream_t)s, n, (const double*)workspace, scale, loss);
  return uh_check_launch("topk_distill_step");
}
