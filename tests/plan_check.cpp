// The page plan's counts (csrc/q36_plan.h) at every pair of a set that holds the borders of an int, against 64 bits.
// Prints each that fails and exits 1.
#include <cstdint>
#include <cstdio>

#define __host__
#define __device__
#define __forceinline__ inline
#include "q36_plan.h"

using namespace q36;

int main() {
  const int counts[] = {0, 1, 2, 3, 4, 15, 16, 17, 1023, 1024, 1025, (1 << 29) - 1, 1 << 29, kMostCount - 1, kMostCount, kMostCount + 1,
                        (1 << 30) - 1024, (1 << 30) - 1, 1 << 30, 2147483646, 2147483647, -1, -2147483647 - 1};
  int bad = 0;
  for (int sh = 0; sh <= 10; ++sh)
    for (int cv : counts)
      for (int nv : counts) {
        const int64_t P = 1 << sh, most = (1 << 30) - (1 << 20);
        const int64_t c = cv < 0 ? 0 : cv < most ? cv : most, n = nv < 0 ? 0 : nv < most ? nv : most;
        const int64_t have = (c + P - 1) / P, full = (c + n + P - 1) / P;
        if (count_of(cv) != c || count_of(nv) != n || c + n > INT32_MAX - (1 << 20)) printf("counts %d %d\n", cv, nv), ++bad;
        else if (pages_of(count_of(cv), sh) != have || pages_of(count_of(cv) + count_of(nv), sh) != full)
          printf("P=%d: %d + %d: %d, %d pages, not %lld, %lld\n", 1 << sh, cv, nv, pages_of(count_of(cv), sh),
                 pages_of(count_of(cv) + count_of(nv), sh), (long long)have, (long long)full), ++bad;
      }
  printf("%d fail\n", bad);
  return bad != 0;
}
