// Keys of attention with a sliding window and sinks, shared by the planner (host) and the
// kernels: both number the keys that a work item reads in the same way.
//
// A query at position i sees the keys j <= i with i - j < window or j < sinks. For rows whose
// first one is at position p, the keys in sight lie in [0, sinks) and from p - window + 1 on.
// The kernels walk them in aligned units of 32 keys, so what is left out is
//   [ns, ns + gap),  ns = sinks rounded up, ns + gap = p - window + 1 rounded down,
// and the others are numbered through: number x is key x below ns, key x + gap from ns on.
// Visible numbers of a row at position i are x <= i - gap with x < sinks or
// x >= i - window + 1 - gap: keys between `sinks` and ns are below every row's window wherever
// gap > 0, so one comparison holds for both sides.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define HY_BOTH __host__ __device__ __forceinline__
#else
#define HY_BOTH inline
#endif

namespace hy {

struct WindowKeys {
  int32_t ns;   // numbers below it are keys of the same number
  int32_t gap;  // keys left out there
};

// sinks <= kMaxSinks, window >= 1, first_pos >= 0.
constexpr int32_t kMaxSinks = 1 << 30;

constexpr int32_t kWindowUnit = 32;

HY_BOTH WindowKeys window_keys(int32_t first_pos, int32_t window, int32_t sinks) {
  const int32_t low = first_pos - window + 1;
  const int32_t from = low > 0 ? low / kWindowUnit * kWindowUnit : 0;
  const int32_t ns = (sinks + kWindowUnit - 1) / kWindowUnit * kWindowUnit;
  return {ns, from > ns ? from - ns : 0};
}

}  // namespace hy
