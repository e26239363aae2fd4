// Log probabilities of given labels, entropy and top alternatives of every row of a table of class logits, and the
// gradient of the first two.  With x a row's logits, T the temperature, z = (x - max x) / T, s = sum e^z, p = e^z / s:
//     log_prob = z[label] - ln s,      entropy H = ln s - (sum e^z z) / s,
//     top: the largest logits (ties: lowest class first) as z - ln s and class
//     dx_j = [ g (delta(j, label) - p_j) - h p_j (ln p_j + H) ] / T        (g, h: gradients of log_prob and H)
#include "class_rows.h"

// ---- one workgroup per row, any strides -------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void label_probs_any_kernel(RowView v, long long rows, const T* __restrict__ x,
                                                              const void* __restrict__ labels, int label_bytes,
                                                              long long ignore, int top, float temperature, float c2,
                                                              float* __restrict__ log_prob, float* __restrict__ entropy,
                                                              float* __restrict__ top_lp, int* __restrict__ top_idx,
                                                              float* __restrict__ stats) {
  __shared__ float fbuf[4];
  __shared__ uint64_t kbuf[4];
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const long long label = labels ? load_int(labels, label_bytes, r) : 0;
    const bool ignored = labels && label == ignore;
    if (ignored) {
      if (threadIdx.x == 0) {
        log_prob[r] = 0.f;
        entropy[r] = 0.f;
        if (stats) { stats[2 * r] = 0.f; stats[2 * r + 1] = INFINITY; }
      }
      for (int k = threadIdx.x; k < top; k += 256) {
        top_lp[v.entry(r, k, top)] = -INFINITY;
        top_idx[v.entry(r, k, top)] = -1;
      }
      continue;
    }
    const T* row = x + v.base(r);
    const RowStat st = block_row_stat(row, v.C, v.sc, c2, fbuf);
    const float ln_s = logf(st.s), m = st.m;
    const bool undefined = !(st.s >= 0.f);
    if (threadIdx.x == 0) {
      entropy[r] = st.s == 0.f ? 0.f : ln_s - (st.t / st.s) * UH_LN2;
      if (labels)
        log_prob[r] = label < 0 || label >= v.C ? NAN
                      : st.s == 0.f             ? -INFINITY
                                                : scaled(ld(row + label * v.sc), m, temperature) - ln_s;
      if (stats) { stats[2 * r] = m; stats[2 * r + 1] = stat_l2(st.s); }
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < top; ++k) {
      uint64_t best = 0;
      if (last && !undefined)
        for (int c = threadIdx.x; c < v.C; c += 256) {
          const uint64_t key = rank_key(ld(row + c * v.sc), c);
          if (key < last && key > best) best = key;
        }
      best = block_max(best, kbuf);
      if (threadIdx.x == 0) {
        top_lp[v.entry(r, k, top)] = undefined ? NAN : best ? scaled(key_value(best), m, temperature) - ln_s : -INFINITY;
        top_idx[v.entry(r, k, top)] = best ? key_class(best) : -1;
      }
      last = best;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void label_probs_bwd_any_kernel(RowView v, RowView vo, long long rows,
                                                                  const T* __restrict__ x, const void* __restrict__ labels,
                                                                  int label_bytes, long long ignore, float inv_t, float c2,
                                                                  const float* __restrict__ stats,
                                                                  const float* __restrict__ entropy,
                                                                  const float* __restrict__ g_lp,
                                                                  const float* __restrict__ g_ent, T* __restrict__ dx) {
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const long long label = labels ? load_int(labels, label_bytes, r) : -1;
    const T* row = x + v.base(r);
    T* out = dx + vo.base(r);
    if (labels && label == ignore) {
      for (int c = threadIdx.x; c < v.C; c += 256) st(out + c * vo.sc, 0.f);
      continue;
    }
    const float m = stats[2 * r], l2 = stats[2 * r + 1];
    const float g = g_lp ? g_lp[r] : 0.f, h = g_ent ? g_ent[r] : 0.f;
    float a = -(g + h * entropy[r]) * inv_t;
    const float b = -h * UH_LN2 * inv_t;
    const float own = l2 == INFINITY ? 0.f : g * inv_t;
    if (g_lp && (label < 0 || label >= v.C)) a = NAN;
    for (int c = threadIdx.x; c < v.C; c += 256) {
      const float l = (ld(row + c * v.sc) - m) * c2 - l2;
      float d = ex2(l) * fmaf(b, fmaxf(l, UH_ZMIN), a);
      if (c == label) d += own;
      st(out + c * vo.sc, d);
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
static unsigned row_grid(long long rows) { return (unsigned)(rows < (1 << 20) ? rows : (1 << 20)); }

extern "C" size_t uh_label_log_probs_workspace(const uh_class_view* view, int top) {
  (void)view;
  (void)top;
  return 0;
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
  UH_REQUIRE(temperature > 0.f && temperature < INFINITY, "label_log_probs: temperature %g", temperature);
  const size_t need = uh_label_log_probs_workspace(view, top);
  UH_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "label_log_probs: workspace of %zu bytes, %zu needed",
             workspace_bytes, need);
  const RowView v = uh_row_view(view);
  const long long rows = v.outer * v.inner;
  const float c2 = (float)(1.4426950408889634 / (double)temperature);
#define UH_GO(T)                                                                                                        \
  hipLaunchKernelGGL(label_probs_any_kernel<T>, dim3(row_grid(rows)), dim3(256), 0, (hipStream_t)s, v, rows,            \
                     (const T*)logits, labels, label_bytes, ignore_index, top, temperature, c2, log_prob, entropy,      \
                     top_log_prob, top_index, stats)
  if (view->dtype == UH_F32) UH_GO(float);
  else if (view->dtype == UH_BF16) UH_GO(bf16);
  else UH_GO(f16);
#undef UH_GO
  return uh_check_launch("label_log_probs");
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
  UH_REQUIRE(temperature > 0.f && temperature < INFINITY, "label_log_probs_bwd: temperature %g", temperature);
  const RowView v = uh_row_view(view), vo = uh_row_view(out_view);
  const long long rows = v.outer * v.inner;
  const float c2 = (float)(1.4426950408889634 / (double)temperature), inv_t = 1.f / temperature;
#define UH_GO(T)                                                                                                        \
  hipLaunchKernelGGL(label_probs_bwd_any_kernel<T>, dim3(row_grid(rows)), dim3(256), 0, (hipStream_t)s, v, vo, rows,    \
                     (const T*)logits, labels, label_bytes, ignore_index, inv_t, c2, stats, entropy, g_log_prob,        \
                     g_entropy, (T*)dlogits)
  if (view->dtype == UH_F32) UH_GO(float);
  else if (view->dtype == UH_BF16) UH_GO(bf16);
  else UH_GO(f16);
#undef UH_GO
  return uh_check_launch("label_log_probs_bwd");
}
