// Distillation from a teacher's top logits.  A row has a student's logits x over C classes and a teacher's slots
// (v_k, i_k), k < K: the logits (or log probabilities: a constant drops out) of a few of its best classes.  With
//     t = softmax over the slots of v / T,     p = softmax over the classes of x / T
//     loss_row = T^2 sum_k t_k (ln t_k - ln p[i_k]),          loss = scale * sum_rows w_row loss_row
//     dx_j = g scale w_row T (p_j - sum_{k: i_k = j} t_k)
// A slot with a negative index is free (t_k = 0).  Rows with w = 0 or without a filled slot count as 0 and get no
// gradient, whatever they hold.  A class index past C or a NaN among a row's slots makes that row's loss and gradient NaN.
#include "class_rows.h"

// teacher's slot k of a row: its value (-inf for a free slot) and class
__device__ __forceinline__ float slot_value(const void* v, int dtype, long long i) {
  return dtype == UH_F32 ? ((const float*)v)[i] : dtype == UH_BF16 ? (float)((const bf16*)v)[i] : (float)((const f16*)v)[i];
}

struct Slots {
  const void* value;
  const void* index;
  int K, dtype, index_bytes;
};

// ---- one workgroup per row, any strides -------------------------------------------------------------------------------
// mode 0: loss only, 1: gradient only (statistics given), 2: both
template <typename T, int MODE>
__global__ __launch_bounds__(256) void distill_any_kernel(RowView v, RowView vo, long long rows, const T* __restrict__ x, Slots sl,
                                                          const float* __restrict__ weight, float temperature, float c2,
                                                          float grad_scale, const float* __restrict__ gout,
                                                          float* __restrict__ stats, float* __restrict__ row_loss,
                                                          T* __restrict__ dx) {
  __shared__ float fbuf[4];
  __shared__ float t_of[UH_SLOTS_MAX];
  __shared__ int i_of[UH_SLOTS_MAX];
  const int tid = threadIdx.x;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const float w = weight ? weight[r] : 1.f;
    const T* row = x + v.base(r);
    __syncthreads();                                   // the slots of the row before are read no more
    // the teacher's softmax: one slot per thread (K <= 256)
    float val = -INFINITY;
    int idx = -1;
    if (tid < sl.K && w != 0.f) {
      const long long e = v.entry(r, tid, sl.K);
      val = slot_value(sl.value, sl.dtype, e);
      const long long i = load_int(sl.index, sl.index_bytes, e);
      idx = i < 0 ? -1 : i >= v.C ? v.C : (int)i;
      if (idx < 0 && val == val) val = -INFINITY;
    }
    const float vm = block_max(val, fbuf);
    const float bad = block_sum((val != val || idx >= v.C) ? 1.f : 0.f, fbuf);
    const bool empty = vm == -INFINITY && bad == 0.f;
    const float ev = val == -INFINITY ? 0.f : ex2((val - vm) * c2);
    const float sv = block_sum(ev, fbuf);
    const float t = bad != 0.f ? NAN : empty ? 0.f : ev / sv;
    if (tid < sl.K) { t_of[tid] = t; i_of[tid] = idx; }
    __syncthreads();
    float m, l2;
    if (empty) {
      m = 0.f, l2 = INFINITY;
    } else if (MODE == 1) {
      m = stats[2 * r], l2 = stats[2 * r + 1];
    } else {
      const RowStat s = block_row_stat(row, v.C, v.sc, c2, fbuf);
      m = s.m, l2 = stat_l2(s.s);
    }
    if (MODE != 1) {
      float part = 0.f;
      if (bad != 0.f) part = NAN;
      else if (t > 0.f) part = t * ((scaled(val, vm, temperature) - logf(sv)) - (scaled(ld(row + idx * v.sc), m, temperature) - l2 * UH_LN2));
      else if (t != t) part = NAN;
      part = block_sum(part, fbuf);
      if (tid == 0) {
        row_loss[r] = empty ? 0.f : w * temperature * temperature * part;
        if (stats) { stats[2 * r] = m; stats[2 * r + 1] = l2; }
      }
    }
    if (MODE != 0) {
      T* out = dx + vo.base(r);
      const float a = empty ? 0.f : (MODE == 1 ? gout[0] * grad_scale : grad_scale) * w * temperature;
      if (empty) {
        for (int c = tid; c < v.C; c += 256) st(out + c * vo.sc, 0.f);
        continue;
      }
      const float sum_t = bad != 0.f || !(sv >= 0.f) ? NAN : 1.f;
      for (int c = tid; c < v.C; c += 256) st(out + c * vo.sc, a * sum_t * ex2((ld(row + c * v.sc) - m) * c2 - l2));
      __syncthreads();                                 // the dense part is written before a slot's class is written again
      if (tid < sl.K && idx >= 0 && idx < v.C) {
        float mine = 0.f;
        for (int k = 0; k < sl.K; ++k) mine += i_of[k] == idx ? t_of[k] : 0.f;
        st(out + idx * vo.sc, a * (sum_t * ex2((ld(row + idx * v.sc) - m) * c2 - l2) - mine));
      }
    }
  }
}

// loss = scale * sum of the rows' losses, in 64 bits and a fixed order
__global__ __launch_bounds__(1024) void distill_finish_kernel(long long n, const float* __restrict__ row_loss, double scale,
                                                              float* __restrict__ loss) {
  __shared__ double buf[1024];
  double a = 0.0;
  for (long long i = threadIdx.x; i < n; i += 1024) a += (double)row_loss[i];
  buf[threadIdx.x] = a;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if (threadIdx.x < o) buf[threadIdx.x] += buf[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) loss[0] = (float)(buf[0] * scale);
}

// ---- host ---------------------------------------------------------------------------------------------------------------
static unsigned row_grid(long long rows) { return (unsigned)(rows < (1 << 20) ? rows : (1 << 20)); }

static int distill_check(const char* who, const uh_class_view* v, const void* logits, const uh_slots* sl, float temperature) {
  const int ok = uh_check_view(v, who);
  if (ok != UH_OK) return ok;
  UH_REQUIRE(sl, "%s: no slots", who);
  UH_REQUIRE(sl->slots > 0 && sl->slots <= UH_SLOTS_MAX, "%s: %d slots (1 to %d)", who, sl->slots, UH_SLOTS_MAX);
  UH_REQUIRE(sl->value_dtype >= UH_F32 && sl->value_dtype <= UH_F16, "%s: slot dtype %d", who, sl->value_dtype);
  UH_REQUIRE(sl->index_bytes == 4 || sl->index_bytes == 8, "%s: slot indices of %d bytes", who, sl->index_bytes);
  UH_REQUIRE(logits && sl->value && sl->index, "%s: null pointer", who);
  UH_REQUIRE(temperature > 0.f && temperature < INFINITY, "%s: temperature %g", who, temperature);
  return UH_OK;
}

static int same_rows(const char* who, const uh_class_view* v, const uh_class_view* o) {
  const int ok = uh_check_view(o, who);
  if (ok != UH_OK) return ok;
  UH_REQUIRE(o->dtype == v->dtype && o->classes == v->classes && o->outer == v->outer && o->inner == v->inner,
             "%s: the gradient's view differs from the logits'", who);
  return UH_OK;
}

template <int MODE>
static void distill_launch(const uh_class_view* view, const uh_class_view* out_view, const void* logits, const uh_slots* s,
                           const float* weight, float temperature, float grad_scale, const float* gout, float* stats,
                           float* row_loss, void* dx, hipStream_t st) {
  const RowView v = uh_row_view(view), vo = uh_row_view(out_view);
  const long long rows = v.outer * v.inner;
  const float c2 = (float)(1.4426950408889634 / (double)temperature);
  const Slots sl{s->value, s->index, s->slots, s->value_dtype, s->index_bytes};
#define UH_GO(T)                                                                                                       \
  hipLaunchKernelGGL((distill_any_kernel<T, MODE>), dim3(row_grid(rows)), dim3(256), 0, st, v, vo, rows,               \
                     (const T*)logits, sl, weight, temperature, c2, grad_scale, gout, stats, row_loss, (T*)dx)
  if (view->dtype == UH_F32) UH_GO(float);
  else if (view->dtype == UH_BF16) UH_GO(bf16);
  else UH_GO(f16);
#undef UH_GO
}

extern "C" size_t uh_topk_distill_workspace(const uh_class_view* view) {
  if (uh_check_view(view, "topk_distill_workspace") != UH_OK) return 0;
  return (size_t)(view->outer * view->inner) * sizeof(float);
}

extern "C" int uh_topk_distill(const uh_class_view* view, const void* logits, const uh_slots* slots, const float* weight,
                               float temperature, double scale, float* loss, float* stats, void* workspace,
                               size_t workspace_bytes, uh_stream s) {
  const int ok = distill_check("topk_distill", view, logits, slots, temperature);
  if (ok != UH_OK) return ok;
  UH_REQUIRE(loss && workspace && workspace_bytes >= uh_topk_distill_workspace(view), "topk_distill: null pointer or workspace of %zu bytes",
             workspace_bytes);
  distill_launch<0>(view, view, logits, slots, weight, temperature, 0.f, nullptr, stats, (float*)workspace, nullptr, (hipStream_t)s);
  hipLaunchKernelGGL(distill_finish_kernel, dim3(1), dim3(1024), 0, (hipStream_t)s, view->outer * view->inner,
                     (const float*)workspace, scale, loss);
  return uh_check_launch("topk_distill");
}

extern "C" int uh_topk_distill_bwd(const uh_class_view* view, const uh_class_view* out_view, const void* logits,
                                   const uh_slots* slots, const float* weight, float temperature, double scale,
                                   const float* gout, const float* stats, void* dlogits, uh_stream s) {
  int ok = distill_check("topk_distill_bwd", view, logits, slots, temperature);
  if (ok == UH_OK) ok = same_rows("topk_distill_bwd", view, out_view);
  if (ok != UH_OK) return ok;
  UH_REQUIRE(gout && stats && dlogits, "topk_distill_bwd: null pointer");
  distill_launch<1>(view, out_view, logits, slots, weight, temperature, (float)scale, gout, const_cast<float*>(stats), nullptr,
                    dlogits, (hipStream_t)s);
  return uh_check_launch("topk_distill_bwd");
}

extern "C" int uh_topk_distill_step(const uh_class_view* view, const uh_class_view* out_view, const void* logits,
                                    const uh_slots* slots, const float* weight, float temperature, double scale,
                                    float grad_scale, float* loss, void* dlogits, void* workspace, size_t workspace_bytes,
                                    uh_stream s) {
  int ok = distill_check("topk_distill_step", view, logits, slots, temperature);
  if (ok == UH_OK) ok = same_rows("topk_distill_step", view, out_view);
  if (ok != UH_OK) return ok;
  UH_REQUIRE(loss && dlogits && workspace && workspace_bytes >= uh_topk_distill_workspace(view),
             "topk_distill_step: null pointer or workspace of %zu bytes", workspace_bytes);
  distill_launch<2>(view, out_view, logits, slots, weight, temperature, (float)(scale * (double)grad_scale), nullptr, nullptr,
                    (float*)workspace, dlogits, (hipStream_t)s);
  hipLaunchKernelGGL(distill_finish_kernel, dim3(1), dim3(1024), 0, (hipStream_t)s, view->outer * view->inner,
                     (const float*)workspace, scale, loss);
  return uh_check_launch("topk_distill_step");
}
