// How the chunk attention deals one call's work to its workgroups: the integer arithmetic, for the kernels and a program
// that checks it over many batches on the CPU.
//
// A tile is a run of new tokens of one request with one KV head's 8 query heads; it walks the keys that its last token
// sees, in steps.  A request of more than kNarrow new tokens is cut into wide tiles (kWideTok tokens, one set of keys for
// all eight waves, kWideKeys a step), another is one narrow tile (up to kNarrow tokens, four sets of keys a step between
// pairs of waves).  The tiles of all requests, head by head, lie on a line; a tile weighs its steps and kTileOvh (what starting
// and ending one costs beside its steps), half before and half behind them.  The line is cut into equal shares, a share a
// workgroup, so that a share holds the end of a tile, whole tiles and the start of another.  A step belongs to the share
// that its place lies in, cuts close to a wide tile's ends apart; a cut tile leaves a partial in each share that has steps of it.
#pragma once
#include <stdint.h>

namespace q36 {

// kNarrow, us a call: 16 requests of 8 tokens behind 500 keys, 4 behind 8000: as narrow tiles 23.5, 28.8, as wide ones 23.0,
// 30.5.  (A narrow tile holds 8 tokens; 12 and 16 as two of them took 10 % longer than as a wide one.)
constexpr int kNarrow = 8, kWideTok = 32, kWideKeys = 32, kNarrowKeys = 128;
// kTileOvh, us a call at 6, 7, 8, 9, 10: eight prompts 45.7, 47.3, 47.2, 48.1, 50.8; 64 requests of 1 .. 200 tokens 21.9, 22.6,
// 22.1, 22.7, 22.0; 24 requests, chunks beside single tokens, 52.9, 53.9, 55.3, 54.7, 56.6; one of 8192 tokens 390 to 393.
// (Chosen when shares joined every cut tile: eight prompts 51.5 at 6, 48.6 at 8.)
constexpr int kTileOvh = 8;
// What a narrow step weighs: it brings 64 KB for a block a wave, a wide one 16.  us a call at 1, 2, 3: 12 requests of 1 .. 300
// tokens over up to 6000 keys 48.5, 41.7, 42.4; 64 of 1 .. 200 21.8, 22.2, 22.2; 24, chunks beside single tokens, 56.0, 55.7, 55.9.
constexpr int kNarrowCost = 2;
// A share is no shorter than a narrow step.  Five tokens over 300 keys at 2, 4, 8, 20: 17.6, 19.0, 20.2, 29.4 us.
constexpr int kLeastShare = kNarrowCost;
// Shares of this length and longer join a tile that two of them cut, where they meet; of shorter ones the second kernel joins
// it, in parallel, while the join, 256 KB read by one workgroup, would make up the call's end.  us a call joined by the shares,
// by the second kernel (share): four chunks of 200 .. 700 tokens 38.6, 34.9 (6), behind 1000 keys 64.5, 59.1 (20), behind 2000
// 83.3, 76.8 (33), behind 4000 115.8, 115.8 (59); prompts: one of 2048 62.0, 58.6 (20), 3000 92.0, 90.6 (40), 4096 131.7, 140.7
// (72), 8192 425, 439 (257); 16 of 64 .. 1000 53.7, 54.7 (25); 8 of 120 .. 2000 77.8, 82.8 (40).
constexpr int kJoinShare = 36;

struct ChunkReq {
  int n, nk;  // new tokens, keys (the new ones included)
};
__host__ __device__ __forceinline__ bool ck_wide(int n) { return n > kNarrow; }
__host__ __device__ __forceinline__ int ck_tiles(int n) { return ck_wide(n) ? (n + kWideTok - 1) / kWideTok : n > 0; }
// the keys that tile i's last token sees
__host__ __device__ __forceinline__ int ck_keys(ChunkReq r, int i) {
  const int end = (i + 1) * kWideTok, k = r.nk - r.n + (end < r.n ? end : r.n);
  return k > 0 ? k : 0;
}
__host__ __device__ __forceinline__ int ck_step_keys(int n) { return ck_wide(n) ? kWideKeys : kNarrowKeys; }
__host__ __device__ __forceinline__ int ck_steps(ChunkReq r, int i) {
  const int ks = ck_step_keys(r.n);
  return (ck_keys(r, i) + ks - 1) / ks;
}
__host__ __device__ __forceinline__ int ck_cost(int n) { return ck_wide(n) ? 1 : kNarrowCost; }
// sum over j < count of max(0, c + j)
__host__ __device__ __forceinline__ int ck_series(int c, int count) {
  if (c < 0) {
    count += c;
    c = 0;
  }
  return count > 0 ? count * c + ((count * (count - 1)) >> 1) : 0;
}
// the weight of one head's tiles before tile i (i up to the number of tiles)
__host__ __device__ __forceinline__ int ck_before(ChunkReq r, int i) {
  int s = i * kTileOvh, full = i;
  if (i == ck_tiles(r.n) && i > 0) {  // the last tile ends with the request
    s += ck_steps(r, i - 1) * ck_cost(r.n);
    --full;
  }
  // the others, of a wide request, see nk - n + kWideTok (k + 1) keys: a step more each
  return s + ck_series(((r.nk - r.n + 31) >> 5) + 1, full);
}
// the weight of a request, both heads (an empty one weighs 1: what passing over it costs)
__host__ __device__ __forceinline__ int ck_weight(ChunkReq r) { return r.n > 0 ? 2 * ck_before(r, ck_tiles(r.n)) : 1; }
// the tile of a head that place x of its line lies in
__host__ __device__ __forceinline__ int ck_tile_at(ChunkReq r, int x) {
  int lo = 0, hi = ck_tiles(r.n) - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (ck_before(r, mid) <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// The most that a call of T new tokens, B requests and tables of `keys` keys can weigh; a line of kMostWeight is not dealt.
constexpr int kMostWeight = 1 << 30;
// the sum of two weights, held there (row starts that are no row starts can count a row for many requests)
__host__ __device__ __forceinline__ int ck_held(int a, int b) {
  const uint32_t s = (uint32_t)a + (uint32_t)b;
  return s < (uint32_t)kMostWeight ? (int)s : kMostWeight;
}
inline bool ck_too_long(int64_t T, int64_t B, int64_t keys) {
  return 2.0 * ((double)T / kWideTok + 2.0 * (double)B) * ((double)keys / kWideKeys + kNarrowCost + kTileOvh) + (double)B >= kMostWeight;
}

// Equal shares: their length, and how many a line has
__host__ __device__ __forceinline__ int ck_share_len(int total, int G) {
  const int len = (total + G - 1) / G;
  return len > kLeastShare ? len : kLeastShare;
}
__host__ __device__ __forceinline__ int ck_shares(int total, int len) { return (total + len - 1) / len; }

// A cut of a wide tile costs some ten steps: its 256 KB leave and come back, and its queries are read twice.  So one that
// falls within kSnap steps of the tile's end goes to that end.  us a call at 0, 3, 4, 5, 6: eight prompts 49.1, 48.8, 47.6, 47.0,
// 46.2; 64 requests of 1 .. 200 tokens 28.5, 22.1, 22.2, 22.1, 22.1; 24, chunks beside single tokens, 52.8, 53.4, 55.4, 56.4, 55.4;
// 2048 tokens behind 6000 191, 190, 190, 189, 194.  A narrow tile's cut stays where it falls: with it moved, without, five tokens
// over 300 keys 18.5, 17.3, four requests of 8 behind 8000 33.2, 28.3, of one over 32000 44.5, 40.0, but 70 of one over 700 24.7,
// 34.4.
// A tile's cuts lie behind step ck_lo and before ck_hi.
constexpr int kSnap = 4;
__host__ __device__ __forceinline__ int ck_lo(int steps, int cost) {
  return cost > 1 ? 0 : kSnap < (steps - 1) / 2 ? kSnap : (steps - 1) / 2;
}
__host__ __device__ __forceinline__ int ck_hi(int steps, int cost) {
  const int lo = ck_lo(steps, cost);
  return cost > 1 ? steps : steps - kSnap > lo + 1 ? steps - kSnap : lo + 1;
}
// The steps [st0, st0 + nst) of a tile at `off` on the line that the share [x0, x1) has; first, last: whether they hold the
// tile's first and last step.  A tile without a step is its start's share's, whole.  nst < 0: the share has none.
struct ChunkRun {
  int st0, nst;
  bool first, last;
};
__host__ __device__ __forceinline__ ChunkRun ck_run(int steps, int cost, int off, int x0, int x1) {
  if (steps == 0) return ChunkRun{0, off >= x0 && off < x1 ? 0 : -1, true, true};
  const int at = off + kTileOvh / 2;  // of its first step
  const int lo = ck_lo(steps, cost), hi = ck_hi(steps, cost);
  int a = x0 > at ? (x0 - at + cost - 1) / cost : 0, e = x1 > at ? (x1 - at + cost - 1) / cost : 0;
  a = a <= lo ? 0 : a >= hi ? steps : a;
  e = e <= lo ? 0 : e >= hi ? steps : e;
  return ChunkRun{a, e > a ? e - a : -1, a == 0, e == steps};
}
// the shares that the first and the last step of a tile at `off` lie in
__host__ __device__ __forceinline__ int ck_first_share(int steps, int cost, int off, int len) {
  return (off + kTileOvh / 2 + ck_lo(steps, cost) * cost) / len;
}
__host__ __device__ __forceinline__ int ck_last_share(int steps, int cost, int off, int len) {
  return (off + kTileOvh / 2 + (ck_hi(steps, cost) - 1) * cost) / len;
}
// The partial of share w: one for a tile that ends here or goes on through, one for a tile that starts here.
__host__ __device__ __forceinline__ int ck_slot(int w, bool first) { return 2 * w + (first ? 1 : 0); }

}  // namespace q36
