#include "scaled_book.cuh"

#include <cuda_fp16.h>
#include <math.h>
#include <string.h>

#include <map>
#include <mutex>

namespace tq {
namespace {

struct Key {
  int n;
  float c[16];
  bool operator<(const Key& o) const { return memcmp(this, &o, sizeof(Key)) < 0; }
};

ScaledBook search(const float* c, int n) {
  ScaledBook sb;
  memset(&sb, 0, sizeof(sb));
  double best = 1e30;
  sb.beta = 1.f;
  for (int step = 0; step < (1 << 16); ++step) {
    const float beta = 1.0f + step * (1.0f / 65536.0f);
    double worst = 0.0;
    for (int i = 0; i < n && worst < best; ++i) {
      if (c[i] == 0.f) continue;
      const double exact = (double)beta * (double)c[i];
      const double rel = fabs((double)__half2float(__float2half_rn((float)exact)) - exact) / fabs(exact);
      if (rel > worst) worst = rel;
    }
    if (worst < best) {
      best = worst;
      sb.beta = beta;
    }
  }
  sb.good = best <= 1.0 / 8192;
  for (int i = 0; i < n; ++i) {
    sb.c16[i] = __half_as_ushort(__float2half_rn(sb.beta * c[i]));
    if (!isfinite(c[i])) sb.good = false;
  }
  return sb;
}

}  // namespace

ScaledBook scaled_book(const float* c, int n) {
  static std::mutex mu;
  static std::map<Key, ScaledBook> kept;
  constexpr size_t kMost = 4096;         // a process that makes codebooks without end does not keep them all
  Key key;
  memset(&key, 0, sizeof(key));
  key.n = n;
  memcpy(key.c, c, n * sizeof(float));
  try {
    std::lock_guard<std::mutex> lock(mu);
    const auto hit = kept.find(key);
    if (hit != kept.end()) return hit->second;
    if (kept.size() >= kMost) kept.clear();
    return kept[key] = search(c, n);
  } catch (...) {                        // no memory to keep it; C callers are above, so nothing may be thrown
    return search(c, n);
  }
}

}  // namespace tq
