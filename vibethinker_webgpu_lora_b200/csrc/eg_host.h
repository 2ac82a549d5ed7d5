// eg_host.h -- internal host helpers shared by eg_host.cpp and eg_runtime.cu.
#pragma once
#include <stdint.h>

#include <atomic>

#include "emberglass.h"

namespace eg {
uint64_t stream_at(uint64_t seed, uint64_t k);
void fill_normal(float* out, int64_t n, uint64_t seed, double stdv, int64_t start);
void rope_tables(int max_ctx, int hd, double theta, float* cosT, float* sinT);
// Records the message for eg_last_error() and returns the status.
eg_status fail(eg_status st, const char* fmt, ...);
// A kernel's launch attribute, set once on each device: first(dev) is true
// until done(dev).  (Twice by two threads at once does no harm.)
struct OncePerDevice {
  std::atomic<uint64_t> seen{0};
  bool first(int dev) const { return dev < 0 || dev > 63 || !(seen.load(std::memory_order_acquire) >> dev & 1); }
  void done(int dev) {
    if (dev >= 0 && dev < 64) seen.fetch_or(1ull << dev, std::memory_order_release);
  }
};
}  // namespace eg
