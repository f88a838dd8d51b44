// The counts of a step's page plan: the integer arithmetic, for the kernel and a program that checks it on the CPU.
#pragma once
#include <stdint.h>

namespace q36 {

// Counts are taken between 0 and this.  A request's keys, its cached and its new ones, then end 2^21 before 2^31, so that a
// thread's walk over them, up to 2^19 at a stride, stays an int to its end.
constexpr int kMostCount = (1 << 30) - (1 << 20);
__host__ __device__ __forceinline__ int count_of(int v) { return v < 0 ? 0 : v < kMostCount ? v : kMostCount; }
// ceil(n / 2^sh), without a sum that passes n.  It grows with n, so a request needs no fewer than zero new pages, and the
// free list's places before a request, sums of those in 64 bits, are none below zero.
__host__ __device__ __forceinline__ int pages_of(int n, int sh) { return (n >> sh) + ((n & ((1 << sh) - 1)) != 0); }

}  // namespace q36
