// Log probabilities of given labels, entropy and top alternatives of every row of a table of class logits, and the
// gradient of the first two.  With x a row's logits, T the temperature, z = (x - max x) / T, s = sum e^z, p = e^z / s:
//     log_prob = z[label] - ln s,      entropy H = ln s - (sum e^z z) / s,
//     top: the largest logits (ties: lowest class first) as z - ln s and class
//     dx_j = [ g (delta(j, label) - p_j) - h p_j (ln p_j + H) ] / T        (g, h: gradients of log_prob and H)
#include "class_rows.h"

struct LpArgs {
  RowView v;
  long long rows;
  const void* labels;
  long long ignore;
  int label_bytes, top;
  float inv_t, c2;
  float *log_prob, *entropy, *top_lp;
  int* top_idx;
  float* stats;
  bool once;                      // uh_read_once

  __device__ __forceinline__ long long label(long long r) const { return labels ? load_int(labels, label_bytes, r) : -1; }
  __device__ __forceinline__ bool ignored(long long l) const { return labels && l == ignore; }
  // by one thread: a row that is not judged; its alternatives are written with write_top(.., 0, ..)
  __device__ __forceinline__ void write_ignored(long long r) const {
    log_prob[r] = 0.f;
    entropy[r] = 0.f;
    if (stats) { stats[2 * r] = 0.f; stats[2 * r + 1] = 0.f; }
  }
  // by one thread: values of a row; x_label: its label's logit where the label is a class.  Returns ln s.
  __device__ __forceinline__ float write_row(long long r, long long l, float x_label, const RowStat& s) const {
    const float ln_s = AnyRef(s.m, c2).ln_s(s.m, s.s);
    // ln s and t share the rounding of M, so that the entropy takes the logarithm of s itself
    entropy[r] = s.s == 0.f ? 0.f : (lg2(s.s) - s.t * rcp(s.s)) * UH_LN2;
    if (labels)
      log_prob[r] = l < 0 || l >= v.C ? NAN : s.s == 0.f ? -INFINITY : scaled(x_label, s.m, inv_t) - ln_s;
    if (stats) { stats[2 * r] = s.m; stats[2 * r + 1] = s.s; }
    return ln_s;
  }
  __device__ __forceinline__ bool is_class(long long l) const { return l >= 0 && l < v.C; }
  // one alternative; cls < 0: the place is left over; undefined rows have s = NaN
  __device__ __forceinline__ void write_top(long long r, int k, float value, int cls, float m, float ln_s, float s) const {
    const bool undefined = !(s >= 0.f);
    const long long e = v.entry(r, k, top);
    top_lp[e] = undefined ? NAN : cls >= 0 ? scaled(value, m, inv_t) - ln_s : -INFINITY;
    top_idx[e] = undefined ? -1 : cls;
  }
};

// ---- rows whose classes lie side by side: 16 or 64 lanes a row, the row in registers -------------------------------------------
// LIST > 0 (G = 16): up to LIST alternatives from the lanes' own falling lists; TOP (G = 64): any number.
// 16 lanes where four loads each hold the row and no more than 8 alternatives are asked for (100000 rows of bf16, 16 and 64 lanes: 300
// classes 17 and 40 us, 512 classes with 1 / 4 / 8 alternatives 46 / 52 / 80 and 97 / 107 / 114 us; 16 lanes with lists of 4 and 8, 300
// classes, top 4: 44.5 and 57.1 us); 64 lanes up to 8 KB, past that a workgroup (bf16, 64
// and 256 lanes: 20000 x 2000 19 and 26 us, 10000 x 4096 with 20 alternatives 39 and 48 us).
template <typename T, int G, int NV, int LIST, bool TOP>
__global__ __launch_bounds__(64) void lp_group_kernel(LpArgs a, const T* __restrict__ x) {
  constexpr int RPB = 64 / G, E = RowRegs<T, G, NV>::E;
  typename Red<G>::Buf red;
  const int C = a.v.C;
  const long long blocks = (a.rows + RPB - 1) / RPB;
  for (long long b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int lane = renew(threadIdx.x % G);
    const long long r = b * RPB + threadIdx.x / G;
    const bool there = r < a.rows;
    const long long l = there ? a.label(r) : 0;
    const bool off = !there || a.ignored(l);
    if (off) {
      if (there) {
        if (lane == 0) a.write_ignored(r);
        for (int k = lane; k < a.top; k += G) a.write_top(r, k, 0.f, -1, 0.f, 0.f, 0.f);
      }
      if (RPB == 1) continue;                              // the whole wave's row
    }
    RowRegs<T, G, NV> reg;
    const T* row = x + (there ? a.v.base(r) : 0);
    if (!off) reg.load(row, 0, C, lane);
    float vmax[TOP ? NV : 1];
    const float lm = off ? -INFINITY : reg.template lane_max<TOP ? NV : 0>(C, vmax);
    RowStat s;
    s.m = group_max<G>(lm);
    if (s.m == -INFINITY) s.m = 0.f;
    reg.fresh();
    group_sums<T, G, NV>(reg, RowRef(s.m, a.c2), C, s, red);
    if (__builtin_expect(__any(is_far(s.m, a.c2)), 0)) {
      RowStat f = s;
      group_sums<T, G, NV>(reg, FarRef(s.m, a.c2), C, f, red);
      if (is_far(s.m, a.c2)) s = f;
    }
    float ln_s = 0.f;
    if (!off) {
      if (lane == 0) ln_s = a.write_row(r, l, a.is_class(l) ? ld(row + l) : 0.f, s);
      else if (LIST > 0 || TOP) ln_s = AnyRef(s.m, a.c2).ln_s(s.m, s.s);
    }
    if constexpr (LIST > 0) {
      TopList<LIST> list;
      reg.fresh();
      if (!off) {
#pragma unroll
        for (int q = 0; q < NV; ++q)
          if (q * G * E < C) {
            const int e = RowRegs<T, G, NV>::first(q, lane, C);
#pragma unroll
            for (int j = 0; j < E; ++j) list.insert(reg.get(q, j), e + j);
          }
      }
      for (int k = 0; k < a.top; ++k) {
        const uint64_t head = list.c[0] < 0 ? 0 : rank_key(list.v[0], list.c[0]);
        const uint64_t best = group_max<G>(head);
        if (best == 0 ? lane == 0 && !off : head == best) {
          a.write_top(r, k, list.v[0], best ? list.c[0] : -1, s.m, ln_s, s.s);
          list.pop();
        }
      }
    }
    if constexpr (TOP) {
      __shared__ TopBuf<G> tb;
      uint32_t low;
      const int found = group_candidates<T, G, NV>(reg, C, lane, 0, a.top, lm, vmax, tb, low);
      const auto emit = [&](int k, uint64_t key) {
        a.write_top(r, k, key_value(key), key ? key_class(key) : -1, s.m, ln_s, s.s);
      };
      if (found <= TopBuf<G>::CAP) group_rank<G>(tb.list, found, lane, a.top, &tb.left, emit);
      else group_rounds<T, G>(row, C, lane, 0, a.top, red, emit);
    }
  }
}

// ---- longer rows: a workgroup of 256 takes a row, or one part of it ----------------------------------------------------------------
// A part leaves its statistics and candidates for the alternatives: all it found, in any order, or the `top` largest where that
// is more than `keep`.  low: order32 of a value that at least `top` of the part's elements reach (0: there are fewer).
// The logits are read once; what bounds it is the exponentials and multiply-adds next to the loads, which hide them only in part
// (a kernel that only reads reaches 6.4 to 7 TB/s here).  bf16: 4096 x 32000 58 us (4.5 TB/s) past the caches, 70 us where a
// backward pass reads them again; 2047 x 50021, top 8: 66 us and 7 to join; 1024 x 131072, top 64: 87 us and 14 to join.
struct LpPart {
  float m, s, t;
  uint32_t low;
  int count, pad[3];
};
// (0 / 16 / 32 / 64 more than `top`: 1024 x 131072 bf16, top 64 106 / 100 / 97.6 / 97.7 us; 4 x 32000, top 20 15.4 / 14.6 / 14.6 / 14.6)
static inline int lp_keep(int top) { return top ? top + 32 : 0; }

template <typename T, int NV, bool TOP>
__global__ __launch_bounds__(256) void lp_rows_kernel(LpArgs a, const T* __restrict__ x, int parts, int part_len, int keep,
                                                      LpPart* __restrict__ part, uint64_t* __restrict__ part_top) {
  __shared__ Red<256>::Buf red;
  const long long r = blockIdx.y + (long long)blockIdx.z * 32768, me = r * parts + blockIdx.x;
  if (r >= a.rows) return;
  const int c0 = blockIdx.x * part_len, lane = threadIdx.x;
  const long long l = a.label(r);
  if (a.ignored(l)) {                                      // (the join does not look at the parts of such a row)
    if (parts == 1) {
      if (lane == 0) a.write_ignored(r);
      for (int k = lane; k < a.top; k += 256) a.write_top(r, k, 0.f, -1, 0.f, 0.f, 0.f);
    }
    return;
  }
  const int n = min(part_len, a.v.C - c0);
  RowRegs<T, 256, NV> reg;
  const T* row = x + a.v.base(r);
  if (a.once) reg.template load<true>(row, c0, n, lane);
  else reg.load(row, c0, n, lane);
  float vmax[TOP ? NV : 1];
  float lm;
  const RowStat s = arriving_stat<T, 256, NV, true, TOP ? NV : 0>(reg, a.c2, n, lm, vmax, red);
  float ln_s = 0.f;
  if (parts == 1) {
    ln_s = AnyRef(s.m, a.c2).ln_s(s.m, s.s);
    if (lane == 0) a.write_row(r, l, a.is_class(l) ? ld(row + l) : 0.f, s);
  }
  uint32_t low = 0;
  int found = 0;
  if constexpr (TOP) {
    __shared__ TopBuf<256> tb;
    found = group_candidates<T, 256, NV>(reg, n, lane, c0, a.top, lm, vmax, tb, low);
    uint64_t* out = part_top + me * keep;
    const auto emit = [&](int k, uint64_t key) {
      if (parts == 1) a.write_top(r, k, key_value(key), key ? key_class(key) : -1, s.m, ln_s, s.s);
      else out[k] = key;
    };
    if (found > TopBuf<256>::CAP) {                        // too many equal values
      group_rounds<T, 256>(row + c0, n, lane, c0, a.top, red, emit);
      found = a.top;                                       // those left over are 0: below any bound
    } else if (parts == 1 || found > keep) {
      group_rank<256>(tb.list, found, lane, a.top, &tb.left, emit);
      found = a.top;
    } else {
      for (int i = lane; i < found; i += 256) out[i] = tb.list[i];
    }
  }
  if (parts == 1) return;
  if (lane == 0) {
    LpPart& p = part[me];
    p.m = s.m, p.s = s.s, p.t = s.t, p.low = low, p.count = found;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void lp_join_kernel(LpArgs a, const T* __restrict__ x, int parts, int keep, const LpPart* __restrict__ part,
                                                      const uint64_t* __restrict__ part_top) {
  extern __shared__ __align__(16) uint64_t keys[];         // parts * keep of them and two to spare
  __shared__ int count, left;
  const long long r = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const long long l = a.label(r);
  if (a.ignored(l)) {
    if (threadIdx.x == 0) a.write_ignored(r);
    for (int k = threadIdx.x; k < a.top; k += 256) a.write_top(r, k, 0.f, -1, 0.f, 0.f, 0.f);
    return;
  }
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  // every wave joins the statistics for itself
  const LpPart* p = part + r * parts + min(lane, parts - 1);
  RowStat s{p->m, p->s, p->t};
  uint32_t low = p->low;
  const int mine = p->count;
  if (lane >= parts) s.s = s.t = 0.f;                      // nobody's part
  for (int o = 1; o < 64 && o < parts; o <<= 1) {
    const RowStat u{__shfl_xor(s.m, o, 64), __shfl_xor(s.s, o, 64), __shfl_xor(s.t, o, 64)};
    s = lane & o ? join(u, s, a.c2) : join(s, u, a.c2);    // the same order of the two in both lanes
    low = max(low, (uint32_t)__shfl_xor(low, o, 64));
  }
  s = RowStat{__shfl(s.m, 0, 64), __shfl(s.s, 0, 64), __shfl(s.t, 0, 64)};
  low = __shfl(low, 0, 64);
  const float ln_s = AnyRef(s.m, a.c2).ln_s(s.m, s.s);
  if (threadIdx.x == 0) a.write_row(r, l, a.is_class(l) ? ld(x + a.v.base(r) + l) : 0.f, s);
  if (a.top == 0) return;
  const uint64_t cut = max((uint64_t)low << 32, (uint64_t)1);
  const uint64_t* from = part_top + r * parts * keep;
  for (int q = threadIdx.x >> 6; q < parts; q += 4) {      // a wave a part
    const int n = __shfl(mine, q, 64);
    for (int i = lane; i < n; i += 64) {
      const uint64_t key = from[q * keep + i];
      if (key >= cut) keys[atomicAdd(&count, 1)] = key;
    }
  }
  __syncthreads();
  group_rank<256>(keys, count, threadIdx.x, a.top, &left, [&](int k, uint64_t key) {
    a.write_top(r, k, key_value(key), key ? key_class(key) : -1, s.m, ln_s, s.s);
  });
}

// ---- one thread per row ----------------------------------------------------------------------------------------------------------
// up to 64 classes in registers (CREG), side by side through LDS (STAGED) or apart.  In 16, 32 and 64 registers: 8 x 16 x 256 x 256
// fp32 8.3, 9.0 and 10.3 us; 8 x 32 x 256 x 256 - , 13.0 and 14.9.  LIST alternatives a sweep: instances of 2, 3, 5 and 8, since
// what a place costs is paid for every class, and those that do not fit for another walk.  8 x 21 x 256 x 256 fp32 with a list of 2 /
// 3 / 5 / 8: top 2 13.5 / 14.1 / 15.7 / 18.2 us, top 3 24.5 / 14.8 / 16.6 / 19.1, top 4 25.5 / 26.9 / 17.5 / 19.8, top 5 37.9 / 27.5 /
// 18.2 / 20.7, top 6 38.4 / 27.8 / 31.4 / 21.2, top 8 51 / 41 / 33 / 22.2, top 9 63 / 42 / 34 / 38.  32 x 21 x 256 x 256 fp32, top 3: 51 us (176 MB read, 50 MB written,
// 4.5 TB/s); 8 x 19 x 251 x 333 16.6 us, gradient 28 us.
template <typename T, int CREG, bool STAGED, int LIST>
__global__ __launch_bounds__(64) void lp_thread_kernel(LpArgs a, const T* __restrict__ x, bool wide) {
  extern __shared__ __align__(16) char lds[];
  T* tile = reinterpret_cast<T*>(lds);
  const int lane = threadIdx.x, C = a.v.C, so = (int)a.v.so;
  const long long blocks = (a.rows + 63) / 64;
  for (long long b = blockIdx.x; b < blocks; b += gridDim.x) {
    const long long r = b * 64 + lane;
    const bool there = r < a.rows;
    if constexpr (STAGED) {
      const int here = (int)min(64ll, a.rows - b * 64);
      __syncthreads();
      copy_to_lds(tile, x + b * 64 * so, (here - 1) * so + C);
      __syncthreads();
    }
    const ApartRows at(a.v, b * 64, lane);
    const auto cls = [&](int c) { return STAGED ? tile + lane * so + c : at.at(x, c * a.v.sc); };
    if (!there) continue;
    float v[CREG];
    if (STAGED && wide) load_classes_wide<T, CREG>(v, tile + lane * so, C);
    else load_classes<T, CREG>(v, C, cls);                                       // on its way while the label is
    const long long l = a.label(r);
    if (a.ignored(l)) {
      a.write_ignored(r);
      for (int k = 0; k < a.top; ++k) a.write_top(r, k, 0.f, -1, 0.f, 0.f, 0.f);
      continue;
    }
    const RowStat s = thread_row_stat<CREG, true>(v, C, a.c2);
    float x_label = 0.f;                                   // apart, 64 labels would be 64 lines: the registers hold them all
    if (STAGED) x_label = a.is_class(l) ? ld(tile + lane * so + (int)l) : 0.f;
    else if (a.labels) {
      const int n = renew_uniform(C);
#pragma unroll
      for (int c = 0; c < CREG; ++c)
        if (c < n) x_label = l == c ? v[c] : x_label;
    }
    const float ln_s = a.write_row(r, l, x_label, s);
    if constexpr (LIST > 0) {
      TopList<LIST> list;
      if constexpr (STAGED || CREG == 64) {                // from LDS or the caches again: 64 unrolled steps cost 256 registers
        for (int c = 0; c < C; ++c) list.insert((float)*cls(c), c);
      } else {
        const int n = renew_uniform(C);
#pragma unroll
        for (int c = 0; c < CREG; ++c)
          if (c < n) list.insert(v[c], c);
      }
      for (int k0 = 0;;) {
#pragma unroll
        for (int i = 0; i < LIST; ++i)
          if (k0 + i < a.top) a.write_top(r, k0 + i, list.v[i], list.c[i], s.m, ln_s, s.s);
        k0 += LIST;
        if (k0 >= a.top) break;
        const float lv = list.v[LIST - 1];                 // the next LIST are those behind the last of these
        const int lc = list.c[LIST - 1];
        list = TopList<LIST>();
        for (int c = 0; c < C; ++c) list.insert(behind((float)*cls(c), c, lv, lc), c);
      }
    }
  }
}

// more classes, lying apart: the thread walks its row, once for the statistics and the first LIST alternatives, and again for
// every LIST more.  8 x 150 x 128 x 128 bf16 with a list of 4 and of 8: top 4 26.6 and 38.0 us, top 5 81.8 and 38.1; without
// alternatives 15.3.
template <typename T, int LIST>
__global__ __launch_bounds__(64) void lp_walk_kernel(LpArgs a, const T* __restrict__ x) {
  const long long r = (long long)blockIdx.x * 64 + threadIdx.x;
  if (r >= a.rows) return;
  const int C = a.v.C;
  const T* row = x + a.v.base(r);
  const long long l = a.label(r);
  if (a.ignored(l)) {
    a.write_ignored(r);
    for (int k = 0; k < a.top; ++k) a.write_top(r, k, 0.f, -1, 0.f, 0.f, 0.f);
    return;
  }
  TopList<LIST ? LIST : 1> list;
  const RowStat s = walk_row_stat(row, a.v.sc, C, a.c2, [&](const float (&v)[16], int c0) {
    if constexpr (LIST > 0)
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (v[j] > list.v[LIST - 1]) list.insert(v[j], c0 + j);
  });
  const float ln_s = a.write_row(r, l, a.is_class(l) ? ld(row + l * a.v.sc) : 0.f, s);
  if constexpr (LIST > 0)
    for (int k0 = 0;;) {
#pragma unroll
      for (int i = 0; i < LIST; ++i)
        if (k0 + i < a.top) a.write_top(r, k0 + i, list.v[i], list.c[i], s.m, ln_s, s.s);
      if ((k0 += LIST) >= a.top) break;
      const float lv = list.v[LIST - 1];                           // more than a list holds: another walk for those behind it
      const int lc = list.c[LIST - 1];
      list = TopList<LIST>();
      for (int c0 = 0; c0 < C; c0 += 8) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c0 + j < C ? ld(row + (c0 + j) * a.v.sc) : -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float u = behind(v[j], c0 + j, lv, lc);
          if (u > list.v[LIST - 1]) list.insert(u, c0 + j);
        }
      }
    }
}

// ---- one workgroup per row, any strides ----------------------------------------------------------------------------------------
template <typename T> __global__ __launch_bounds__(256) void lp_any_kernel(LpArgs a, const T* __restrict__ x) {
  __shared__ Red<256>::Buf red;
  const int lane = threadIdx.x, C = a.v.C;
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const long long l = a.label(r);
    if (a.ignored(l)) {
      if (lane == 0) a.write_ignored(r);
      for (int k = lane; k < a.top; k += 256) a.write_top(r, k, 0.f, -1, 0.f, 0.f, 0.f);
      continue;
    }
    const T* row = x + a.v.base(r);
    const RowStat s = strided_row_stat<T, 256>(row, C, a.v.sc, a.c2, lane, red);
    float ln_s = 0.f;
    if (lane == 0) ln_s = a.write_row(r, l, a.is_class(l) ? ld(row + l * a.v.sc) : 0.f, s);
    uint64_t last = ~0ull;
    for (int k = 0; k < a.top; ++k) {
      uint64_t best = 0;
      for (int c = lane; c < C; c += 256) {
        const uint64_t key = rank_key(ld(row + c * a.v.sc), c);
        if (key < last && key > best) best = key;
      }
      best = Red<256>::maxkey(best, red);
      if (lane == 0) a.write_top(r, k, key_value(best), best ? key_class(best) : -1, s.m, ln_s, s.s);
      last = best;
    }
  }
}

// ---- gradient ---------------------------------------------------------------------------------------------------------------------
struct LpBwd {
  RowView v, vo;
  long long rows;
  const void* labels;
  long long ignore;
  int label_bytes;
  float inv_t, c2;
  const float *stats, *entropy, *g_lp, *g_ent;
};
// One pass: the row is read, its gradient written (4096 x 32000 bf16: 525 MB, 84 us, 6.2 TB/s, what a copy reaches).  The walk of
// classes that lie apart: 8 x 150 x 128 x 128 bf16 25 us.
// dx = e (b z + a) with e = 2^z, z = c x - M: the row's 1/s and ln s are folded into a and b
struct LpCoef {
  float a, b, own, m;
  int label;              // -1: none
  bool off;
  __device__ __forceinline__ LpCoef(const LpBwd& k, long long r) {
    const long long l = k.labels ? load_int(k.labels, k.label_bytes, r) : -1;
    off = k.labels && l == k.ignore;
    m = k.stats[2 * r];
    const float s = k.stats[2 * r + 1];
    const float g = k.g_lp ? k.g_lp[r] : 0.f, h = k.g_ent ? k.g_ent[r] : 0.f;
    const float l2 = lg2(s), inv = rcp(s);
    const bool bad = k.g_lp && (l < 0 || l >= k.v.C);
    b = -h * UH_LN2 * k.inv_t;
    a = bad ? NAN : (-(g + h * k.entropy[r]) * k.inv_t - b * l2) * inv;
    b *= inv;
    own = g * k.inv_t;
    label = l >= 0 && l < k.v.C && k.g_lp ? (int)l : -1;
    if (s == 0.f || off) a = b = own = 0.f, label = -1;
  }
  template <typename R> __device__ __forceinline__ float of(const R& ref, float x) const {
    const float z = ref.z(x);
    return ex2(z) * fmaf(b, fmaxf(z, UH_ZMIN), a);
  }
};

template <typename T, int G, int NV>
__global__ __launch_bounds__(G > 64 ? G : 64) void lp_bwd_group_kernel(LpBwd k, const T* __restrict__ x, T* __restrict__ dx, int part_len) {
  constexpr int RPB = G > 64 ? 1 : 64 / G;
  const int c0 = blockIdx.y * part_len;
  const int n = min(part_len, k.v.C - c0);
  const long long blocks = (k.rows + RPB - 1) / RPB;
  for (long long b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int lane = renew(threadIdx.x % G);
    const long long r = b * RPB + threadIdx.x / G;
    if (r >= k.rows) continue;
    const LpCoef q(k, r);
    T* out = dx + k.vo.base(r);
    RowRegs<T, G, NV> reg;
    if (q.off) {
      reg.map_store(out, c0, n, lane, [](float) { return 0.f; });
      continue;
    }
    const T* row = x + k.v.base(r);
    reg.load(row, c0, n, lane);
    with_ref(q.m, k.c2, [&](const auto& ref) { reg.map_store(out, c0, n, lane, [&](float v) { return q.of(ref, v); }); });
    // the label's class once more, by the lane that has just written it
    const int at = q.label - c0;
    if (at >= 0 && at < n && (at / RowRegs<T, G, NV>::E) % G == lane)
      st(out + q.label, q.of(AnyRef(q.m, k.c2), ld(row + q.label)) + q.own);
  }
}

// up to 64 classes, rows side by side in both tensors
template <typename T> __global__ __launch_bounds__(64) void lp_bwd_thread_kernel(LpBwd k, const T* __restrict__ x, T* __restrict__ dx, bool wide) {
  extern __shared__ __align__(16) char lds[];
  constexpr int E = 16 / sizeof(T);
  const int lane = threadIdx.x, C = k.v.C, so = (int)k.v.so;
  T* tile = reinterpret_cast<T*>(lds);
  T* res = tile + (64 * so + E - 1) / E * E;
  const long long blocks = (k.rows + 63) / 64;
  for (long long b = blockIdx.x; b < blocks; b += gridDim.x) {
    const long long r = b * 64 + lane;
    const int here = (int)min(64ll, k.rows - b * 64);
    __syncthreads();
    copy_to_lds(tile, x + b * 64 * so, (here - 1) * so + C);
    __syncthreads();
    if (lane < here) {
      const LpCoef q(k, r);
      const T* row = tile + lane * so;
      T* out = res + lane * C;
      if (q.off) {
        for (int c = 0; c < C; ++c) out[c] = (T)0.f;
      } else {
        with_ref(q.m, k.c2, [&](const auto& ref) {
          if (wide) {                                      // C and so multiples of 16 bytes
            for (int c = 0; c < C; c += E) {
              alignas(16) T v[E];
              *reinterpret_cast<Vec16*>(v) = *reinterpret_cast<const Vec16*>(row + c);
#pragma unroll
              for (int j = 0; j < E; ++j) v[j] = (T)(q.of(ref, (float)v[j]) + (c + j == q.label ? q.own : 0.f));
              *reinterpret_cast<Vec16*>(out + c) = *reinterpret_cast<const Vec16*>(v);
            }
          } else {
            for (int c = 0; c < C; ++c) out[c] = (T)(q.of(ref, (float)row[c]) + (c == q.label ? q.own : 0.f));
          }
        });
      }
    }
    __syncthreads();
    copy_from_lds(dx + b * 64 * C, res, here * C);
  }
}

// up to 64 classes that lie apart
template <typename T> __global__ __launch_bounds__(64) void lp_bwd_apart_kernel(LpBwd k, const T* __restrict__ x, T* __restrict__ dx) {
  const int lane = threadIdx.x, C = k.v.C;
  const long long blocks = (k.rows + 63) / 64;
  for (long long b = blockIdx.x; b < blocks; b += gridDim.x) {
    const long long r = b * 64 + lane;
    const ApartRows at(k.v, b * 64, lane), to(k.vo, b * 64, lane);
    if (r >= k.rows) continue;
    const LpCoef q(k, r);
    with_ref(q.m, k.c2, [&](const auto& ref) {
      for (int c0 = 0; c0 < C; c0 += 16) {
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c0 + j < C) v[j] = (float)*at.at(x, (c0 + j) * k.v.sc);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c0 + j < C) *to.at(dx, (c0 + j) * k.vo.sc) = (T)(q.off ? 0.f : q.of(ref, v[j]) + (c0 + j == q.label ? q.own : 0.f));
      }
    });
  }
}

// classes that lie apart: one thread per row
template <typename T> __global__ __launch_bounds__(64) void lp_bwd_walk_kernel(LpBwd k, const T* __restrict__ x, T* __restrict__ dx) {
  const long long r = (long long)blockIdx.x * 64 + threadIdx.x;
  if (r >= k.rows) return;
  const LpCoef q(k, r);
  const AnyRef ref(q.m, k.c2);
  const T* row = x + k.v.base(r);
  T* out = dx + k.vo.base(r);
  const int C = k.v.C;
  constexpr int N = 16;                                              // a turn; the next ones are on their way
  T next[N];
  auto fetch = [&](int c0) {
#pragma unroll
    for (int j = 0; j < N; ++j) next[j] = c0 + j < C && !q.off ? row[(c0 + j) * k.v.sc] : (T)0.f;
  };
  fetch(0);
  for (int c0 = 0; c0 < C; c0 += N) {
    float v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (float)next[j];
    if (c0 + N < C) fetch(c0 + N);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (c0 + j < C) st(out + (c0 + j) * k.vo.sc, q.off ? 0.f : q.of(ref, v[j]) + (c0 + j == q.label ? q.own : 0.f));
  }
}

// one workgroup per row, any strides
template <typename T> __global__ __launch_bounds__(256) void lp_bwd_any_kernel(LpBwd k, const T* __restrict__ x, T* __restrict__ dx) {
  for (long long r = blockIdx.x; r < k.rows; r += gridDim.x) {
    const LpCoef q(k, r);
    const AnyRef ref(q.m, k.c2);
    const T* row = x + k.v.base(r);
    T* out = dx + k.vo.base(r);
    for (int c = threadIdx.x; c < k.v.C; c += 256)
      st(out + c * k.vo.sc, q.off ? 0.f : q.of(ref, ld(row + c * k.v.sc)) + (c == q.label ? q.own : 0.f));
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------
// How the rows of a forward call are cut (one part: they are not).  With alternatives parts are 32 KB: looking for candidates
// is what a workgroup's other waves wait for, and 68 registers leave room for seven workgroups a CU, 108 for four (1024 rows
// of 131072 bf16 classes, top 64: 110 us from 64 KB, 105 us from 32 KB).  Without, 64 KB: fewer parts to join.
static RowCut lp_cut(const RowView& v, long long rows, int dtype, int top) {
  if (uh_class_path(v, nullptr, rows, dtype) != PATH_GROUP || (long long)v.C * uh_elem_bytes(dtype) <= 8192) return RowCut{1, v.C};
  return uh_row_cut(rows, v.C, dtype, top ? 32768 : 65536);
}

extern "C" size_t uh_label_log_probs_workspace(const uh_class_view* view, int top) {
  if (uh_check_view(view, "label_log_probs_workspace") != UH_OK || top < 0 || top > UH_TOP_MAX) return 0;
  const long long rows = view->outer * view->inner;
  const int parts = lp_cut(uh_row_view(view), rows, view->dtype, top).parts;
  if (parts == 1) return 0;
  return (size_t)rows * parts * (sizeof(LpPart) + 8 * (size_t)lp_keep(top));
}

template <typename T> static void lp_launch(const LpArgs& a, const T* x, int dtype, void* ws, hipStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const int C = a.v.C;
  const long long rows = a.rows;
  const ClassPath path = uh_class_path(a.v, nullptr, rows, dtype);
  const dim3 waves(uh_grid((rows + 63) / 64, UH_GRID_WAVES));
  if (path == PATH_STAGED || path == PATH_APART) {
    const bool staged = path == PATH_STAGED, wide = staged && (a.v.so * sizeof(T)) % 16 == 0;
    const size_t lds = staged ? (size_t)64 * a.v.so * sizeof(T) : 0;
#define UH_GO3(R, ST, LI) hipLaunchKernelGGL((lp_thread_kernel<T, R, ST, LI>), waves, dim3(64), lds, s, a, x, wide)
#define UH_GO2(R, ST) do { if (a.top == 0) UH_GO3(R, ST, 0); else if (a.top <= 2) UH_GO3(R, ST, 2); else if (a.top == 3) UH_GO3(R, ST, 3); else if (a.top <= 5) UH_GO3(R, ST, 5); else UH_GO3(R, ST, 8); } while (0)
#define UH_GO(ST) do { if (C <= 16) UH_GO2(16, ST); else if (C <= 32) UH_GO2(32, ST); else UH_GO2(64, ST); } while (0)
    if (staged) UH_GO(true); else UH_GO(false);
#undef UH_GO
#undef UH_GO2
#undef UH_GO3
  } else if (path == PATH_WALK) {
    const dim3 grid((unsigned)((rows + 63) / 64));
    if (a.top == 0) hipLaunchKernelGGL((lp_walk_kernel<T, 0>), grid, dim3(64), 0, s, a, x);
    else if (a.top <= 4) hipLaunchKernelGGL((lp_walk_kernel<T, 4>), grid, dim3(64), 0, s, a, x);
    else hipLaunchKernelGGL((lp_walk_kernel<T, 8>), grid, dim3(64), 0, s, a, x);
  } else if (path == PATH_ANY) {
    hipLaunchKernelGGL((lp_any_kernel<T>), dim3(uh_grid(rows, UH_GRID_WAVES)), dim3(256), 0, s, a, x);
  } else if (C <= 16 * 4 * E && a.top <= 8) {
    const dim3 quads(uh_grid((rows + 3) / 4, UH_GRID_WAVES));
    if (a.top == 0) hipLaunchKernelGGL((lp_group_kernel<T, 16, 4, 0, false>), quads, dim3(64), 0, s, a, x);
    else if (a.top <= 4) hipLaunchKernelGGL((lp_group_kernel<T, 16, 4, 4, false>), quads, dim3(64), 0, s, a, x);
    else hipLaunchKernelGGL((lp_group_kernel<T, 16, 4, 8, false>), quads, dim3(64), 0, s, a, x);
  } else if (C <= 64 * 8 * E) {
    const dim3 blocks(uh_grid(rows, UH_GRID_WAVES));
#define UH_GO(NV)                                                                                               \
  do {                                                                                                          \
    if (a.top) hipLaunchKernelGGL((lp_group_kernel<T, 64, NV, 0, true>), blocks, dim3(64), 0, s, a, x);         \
    else hipLaunchKernelGGL((lp_group_kernel<T, 64, NV, 0, false>), blocks, dim3(64), 0, s, a, x);              \
  } while (0)
    if (C <= 64 * 4 * E) UH_GO(4); else UH_GO(8);
#undef UH_GO
  } else {
    const RowCut cut = lp_cut(a.v, rows, dtype, a.top);
    const int keep = lp_keep(a.top);
    LpPart* ps = (LpPart*)ws;
    uint64_t* pt = (uint64_t*)(ps + (size_t)rows * cut.parts);
    const dim3 grid((unsigned)cut.parts, (unsigned)(rows < 32768 ? rows : 32768), (unsigned)((rows + 32767) / 32768));
#define UH_GO(NV, TOP) hipLaunchKernelGGL((lp_rows_kernel<T, NV, TOP>), grid, dim3(256), 0, s, a, x, cut.parts, cut.len, keep, ps, pt)
#define UH_GO2(NV) do { if (a.top) UH_GO(NV, true); else UH_GO(NV, false); } while (0)
    // parts of 32 bits are longer than 1024 classes; with alternatives longer than 32 KB only where 64 of those are not enough
    // (more than 524288 classes of 32 bits)
    if (cut.len <= 256 * 4 * E) {
      if constexpr (sizeof(T) == 2) { if (cut.len <= 256 * E) UH_GO2(1); else UH_GO2(4); }
      else UH_GO2(4);
    } else if (cut.len <= 256 * 8 * E) UH_GO2(8);
    else if constexpr (sizeof(T) == 2) UH_GO(16, false);
    else UH_GO2(16);
#undef UH_GO2
#undef UH_GO
    if (cut.parts > 1)
      hipLaunchKernelGGL((lp_join_kernel<T>), dim3((unsigned)rows), dim3(256), ((size_t)cut.parts * keep + 2) * 8, s, a, x, cut.parts,
                         keep, ps, pt);
  }
}

extern "C" int uh_label_log_probs(const uh_class_view* view, const void* logits, const void* labels, int label_bytes,
                                  long long ignore_index, int top, float temperature, float* log_prob, float* entropy,
                                  float* top_log_prob, int* top_index, float* stats, void* workspace,
                                  size_t workspace_bytes, uh_stream s) {
  const int ok = uh_check_view(view, "label_log_probs");
  if (ok != UH_OK) return ok;
  UH_REQUIRE(logits && entropy, "label_log_probs: null pointer");
  UH_REQUIRE(!labels || (log_prob && (label_bytes == 4 || label_bytes == 8)), "label_log_probs: labels of %d bytes, log_prob %p",
             label_bytes, (void*)log_prob);
  UH_REQUIRE(top >= 0 && top <= UH_TOP_MAX && top <= view->classes, "label_log_probs: top=%d of %d classes (at most %d)", top,
             view->classes, UH_TOP_MAX);
  UH_REQUIRE(top == 0 || (top_log_prob && top_index), "label_log_probs: null pointer");
  UH_REQUIRE(uh_temperature(temperature), "label_log_probs: temperature %g (1e-6 to 1e6)", temperature);
  const size_t need = uh_label_log_probs_workspace(view, top);
  UH_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
             "label_log_probs: workspace of %zu bytes, %zu needed on 16 bytes", workspace_bytes, need);
  LpArgs a;
  a.v = uh_row_view(view);
  a.rows = view->outer * view->inner;
  a.labels = labels, a.label_bytes = label_bytes, a.ignore = ignore_index;
  a.top = top, a.inv_t = 1.f / temperature, a.c2 = (float)(1.4426950408889634 / (double)temperature);
  a.log_prob = log_prob, a.entropy = entropy, a.top_lp = top_log_prob, a.top_idx = top_index, a.stats = stats;
  a.once = uh_read_once(a.v, a.rows, view->dtype, stats);
  if (view->dtype == UH_F32) lp_launch<float>(a, (const float*)logits, view->dtype, workspace, (hipStream_t)s);
  else if (view->dtype == UH_BF16) lp_launch<bf16>(a, (const bf16*)logits, view->dtype, workspace, (hipStream_t)s);
  else lp_launch<f16>(a, (const f16*)logits, view->dtype, workspace, (hipStream_t)s);
  return uh_check_launch("label_log_probs");
}

template <typename T> static void lp_bwd_launch(const LpBwd& k, const T* x, T* dx, int dtype, hipStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const int C = k.v.C;
  const long long rows = k.rows;
  const ClassPath path = uh_class_path(k.v, &k.vo, rows, dtype);
  if (path == PATH_STAGED) {
    const bool wide = (k.v.so * sizeof(T)) % 16 == 0 && (C * sizeof(T)) % 16 == 0;
    const size_t lds = ((64 * k.v.so + E - 1) / E * E + 64 * C) * sizeof(T);
    hipLaunchKernelGGL((lp_bwd_thread_kernel<T>), dim3(uh_grid((rows + 63) / 64, UH_GRID_WAVES)), dim3(64), lds, s, k, x, dx, wide);
  } else if (path == PATH_APART) {
    hipLaunchKernelGGL((lp_bwd_apart_kernel<T>), dim3(uh_grid((rows + 63) / 64, UH_GRID_WAVES)), dim3(64), 0, s, k, x, dx);
  } else if (path == PATH_WALK) {
    hipLaunchKernelGGL((lp_bwd_walk_kernel<T>), dim3((unsigned)((rows + 63) / 64)), dim3(64), 0, s, k, x, dx);
  } else if (path == PATH_ANY) {
    hipLaunchKernelGGL((lp_bwd_any_kernel<T>), dim3(uh_grid(rows, UH_GRID_WAVES)), dim3(256), 0, s, k, x, dx);
  } else if (C <= 16 * 4 * E) {
    hipLaunchKernelGGL((lp_bwd_group_kernel<T, 16, 4>), dim3(uh_grid((rows + 3) / 4, UH_GRID_WAVES)), dim3(64), 0, s, k, x, dx, C);
  } else if (C <= 64 * 4 * E) {
    hipLaunchKernelGGL((lp_bwd_group_kernel<T, 64, 4>), dim3(uh_grid(rows, UH_GRID_WAVES)), dim3(64), 0, s, k, x, dx, C);
  } else {
    const RowCut cut = uh_cut_parts(C, (C + 256 * 4 * E - 1) / (256 * 4 * E));
    hipLaunchKernelGGL((lp_bwd_group_kernel<T, 256, 4>), dim3(uh_grid(rows, UH_GRID_WAVES), (unsigned)cut.parts), dim3(256), 0, s, k,
                       x, dx, cut.len);
  }
}

extern "C" int uh_label_log_probs_bwd(const uh_class_view* view, const uh_class_view* out_view, const void* logits,
                                      const void* labels, int label_bytes, long long ignore_index, float temperature,
                                      const float* stats, const float* entropy, const float* g_log_prob,
                                      const float* g_entropy, void* dlogits, uh_stream s) {
  int ok = uh_check_view(view, "label_log_probs_bwd");
  if (ok == UH_OK) ok = uh_check_view(out_view, "label_log_probs_bwd");
  if (ok != UH_OK) return ok;
  UH_REQUIRE(out_view->dtype == view->dtype && out_view->classes == view->classes && out_view->outer == view->outer &&
                 out_view->inner == view->inner,
             "label_log_probs_bwd: the gradient's view differs from the logits'");
  UH_REQUIRE(logits && stats && entropy && dlogits, "label_log_probs_bwd: null pointer");
  UH_REQUIRE(!labels || label_bytes == 4 || label_bytes == 8, "label_log_probs_bwd: labels of %d bytes", label_bytes);
  UH_REQUIRE(labels || !g_log_prob, "label_log_probs_bwd: a gradient of log_prob without labels");
  UH_REQUIRE(uh_temperature(temperature), "label_log_probs_bwd: temperature %g (1e-6 to 1e6)", temperature);
  LpBwd k;
  k.v = uh_row_view(view), k.vo = uh_row_view(out_view);
  k.rows = view->outer * view->inner;
  k.labels = labels, k.label_bytes = label_bytes, k.ignore = ignore_index;
  k.inv_t = 1.f / temperature, k.c2 = (float)(1.4426950408889634 / (double)temperature);
  k.stats = stats, k.entropy = entropy, k.g_lp = g_log_prob, k.g_ent = g_entropy;
  if (view->dtype == UH_F32) lp_bwd_launch<float>(k, (const float*)logits, (float*)dlogits, view->dtype, (hipStream_t)s);
  else if (view->dtype == UH_BF16) lp_bwd_launch<bf16>(k, (const bf16*)logits, (bf16*)dlogits, view->dtype, (hipStream_t)s);
  else lp_bwd_launch<f16>(k, (const f16*)logits, (f16*)dlogits, view->dtype, (hipStream_t)s);
  return uh_check_launch("label_log_probs_bwd");
}
