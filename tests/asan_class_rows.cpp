// Host-side walk through the entry points over class logits under AddressSanitizer (built by `make -C unet_amd/csrc asan_class_rows`).
// No GPU is needed: workspace sizes are pure host functions, and every other call is refused before anything is launched.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <thread>
#include <vector>

#include "unet_hip.h"

static int failures = 0;
#define EXPECT(cond)                                                          \
  do {                                                                        \
    if (!(cond)) {                                                            \
      std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond);           \
      ++failures;                                                             \
    }                                                                         \
  } while (0)

static void refuse(int status, const char* needle) {
  EXPECT(status != UH_OK);
  const char* msg = uh_last_error();
  EXPECT(msg && std::strlen(msg) > 0 && std::strlen(msg) < 512 && std::strstr(msg, needle) != nullptr);
}

// sizes: every path and border of the rules that cut rows into parts
static void sizes() {
  for (int dtype : {UH_F32, UH_BF16, UH_F16})
    for (int c : {1, 2, 16, 63, 64, 65, 512, 513, 2048, 2049, 4096, 4097, 16384, 16385, 40000, 131072, (int)UH_CLASSES_MAX})
      for (long long rows : {1ll, 3ll, 511ll, 512ll, 4096ll, 4097ll, 1ll << 20, 0x7fffffffll})
        for (int layout = 0; layout < 4; ++layout) {
          uh_class_view v{rows, 1, c, 0, 1, c, dtype};
          if (layout == 1) v.so = c + 13;
          if (layout == 2) v = {1, rows, rows * c, 1, rows, c, dtype};
          if (layout == 3) v = {rows, 1, 0, 0, 0, c, dtype};
          const bool long_rows = v.sc == 1 && c > 64 && (long long)c * (dtype == UH_F32 ? 4 : 2) > 8192;
          const size_t plain = uh_label_log_probs_workspace(&v, 0);
          for (int top : {1, 20, (int)UH_TOP_MAX}) {
            if (top > c) continue;
            const size_t with = uh_label_log_probs_workspace(&v, top);
            EXPECT(with >= plain && with % rows == 0 && (long_rows || with == 0));
          }
          EXPECT(uh_label_log_probs_workspace(&v, -1) == 0 && uh_label_log_probs_workspace(&v, UH_TOP_MAX + 1) == 0);
          EXPECT(uh_topk_distill_workspace(&v) >= 8192 * sizeof(double));
        }
}

static void refusals() {
  char buf[256] = {};
  void* p = buf;                        // never dereferenced: validation fails first
  float* f = (float*)p;
  const uh_class_view ok{4, 1, 6, 0, 1, 6, UH_F32}, other{4, 1, 7, 0, 1, 7, UH_F32};
  const uh_slots slots{p, p, 3, UH_F32, 4};
  for (uh_class_view bad : {uh_class_view{0, 1, 6, 0, 1, 6, UH_F32}, uh_class_view{4, 0, 6, 0, 1, 6, UH_F32}, uh_class_view{4, 1, 6, 0, 1, 0, UH_F32},
                            uh_class_view{4, 1, 6, 0, 1, UH_CLASSES_MAX + 1, UH_F32}, uh_class_view{4, 1, 6, 0, 1, 6, 3},
                            uh_class_view{4, 1, -6, 0, 1, 6, UH_F32}, uh_class_view{1 << 20, 1 << 20, 6, 0, 1, 6, UH_F32}}) {
    EXPECT(uh_label_log_probs_workspace(&bad, 0) == 0 && uh_topk_distill_workspace(&bad) == 0);
    refuse(uh_label_log_probs(&bad, p, p, 8, -100, 0, 1.f, f, f, nullptr, nullptr, nullptr, nullptr, 0, nullptr), "label_log_probs");
    refuse(uh_label_log_probs_bwd(&ok, &bad, p, p, 8, -100, 1.f, f, f, f, f, p, nullptr), "label_log_probs_bwd");
    refuse(uh_topk_distill(&bad, p, &slots, nullptr, 1.f, 1.0, f, nullptr, p, 256, nullptr), "topk_distill");
    refuse(uh_topk_distill_bwd(&ok, &bad, p, &slots, nullptr, 1.f, 1.0, f, f, p, nullptr), "topk_distill_bwd");
    refuse(uh_topk_distill_step(&bad, &ok, p, &slots, nullptr, 1.f, 1.0, 1.f, f, p, p, 256, nullptr), "topk_distill_step");
  }
  for (float t : {0.f, -1.f, 5e-7f, 2e6f, (float)NAN, (float)INFINITY}) {
    refuse(uh_label_log_probs(&ok, p, p, 8, -100, 0, t, f, f, nullptr, nullptr, nullptr, nullptr, 0, nullptr), "temperature");
    refuse(uh_label_log_probs_bwd(&ok, &ok, p, p, 8, -100, t, f, f, f, f, p, nullptr), "temperature");
    refuse(uh_topk_distill(&ok, p, &slots, nullptr, t, 1.0, f, nullptr, p, 256, nullptr), "temperature");
    refuse(uh_topk_distill_bwd(&ok, &ok, p, &slots, nullptr, t, 1.0, f, f, p, nullptr), "temperature");
    refuse(uh_topk_distill_step(&ok, &ok, p, &slots, nullptr, t, 1.0, 1.f, f, p, p, 256, nullptr), "temperature");
  }
  refuse(uh_label_log_probs(&ok, p, p, 8, -100, 7, 1.f, f, f, f, (int*)p, nullptr, nullptr, 0, nullptr), "top=7");
  refuse(uh_label_log_probs(&ok, p, p, 3, -100, 0, 1.f, f, f, nullptr, nullptr, nullptr, nullptr, 0, nullptr), "labels of 3 bytes");
  refuse(uh_label_log_probs_bwd(&ok, &other, p, p, 8, -100, 1.f, f, f, f, f, p, nullptr), "differs");
  refuse(uh_label_log_probs_bwd(&ok, &ok, p, nullptr, 0, -100, 1.f, f, f, f, f, p, nullptr), "without labels");
  const uh_class_view cut{2, 1, 131072, 0, 1, 131072, UH_BF16};
  const size_t need = uh_label_log_probs_workspace(&cut, 5);
  EXPECT(need > 0);
  refuse(uh_label_log_probs(&cut, p, p, 8, -100, 5, 1.f, f, f, f, (int*)p, nullptr, nullptr, need, nullptr), "workspace");
  refuse(uh_label_log_probs(&cut, p, p, 8, -100, 5, 1.f, f, f, f, (int*)p, nullptr, p, need - 1, nullptr), "workspace");
  for (uh_slots bad : {uh_slots{p, p, 0, UH_F32, 4}, uh_slots{p, p, UH_SLOTS_MAX + 1, UH_F32, 4}, uh_slots{p, p, 3, 7, 4}, uh_slots{p, p, 3, UH_F32, 2},
                       uh_slots{nullptr, p, 3, UH_F32, 4}, uh_slots{p, nullptr, 3, UH_F32, 8}}) {
    refuse(uh_topk_distill(&ok, p, &bad, nullptr, 1.f, 1.0, f, nullptr, p, 256, nullptr), "topk_distill");
    refuse(uh_topk_distill_bwd(&ok, &ok, p, &bad, nullptr, 1.f, 1.0, f, f, p, nullptr), "topk_distill_bwd");
    refuse(uh_topk_distill_step(&ok, &ok, p, &bad, nullptr, 1.f, 1.0, 1.f, f, p, p, 256, nullptr), "topk_distill_step");
  }
  refuse(uh_topk_distill(&ok, p, &slots, nullptr, 1.f, 1.0, f, nullptr, p, uh_topk_distill_workspace(&ok) - 1, nullptr), "workspace");
  refuse(uh_topk_distill_step(&ok, &other, p, &slots, nullptr, 1.f, 1.0, 1.f, f, p, p, 1 << 20, nullptr), "differs");
  refuse(uh_topk_distill_bwd(&ok, &ok, p, &slots, nullptr, 1.f, 1.0, nullptr, f, p, nullptr), "null");
}

int main() {
  sizes();
  refusals();
  std::vector<std::thread> threads;     // the error text is each thread's own
  for (int i = 0; i < 4; ++i) threads.emplace_back(refusals);
  for (auto& t : threads) t.join();
  if (!failures) std::printf("class rows under ASan: ok\n");
  return failures ? 1 : 0;
}
