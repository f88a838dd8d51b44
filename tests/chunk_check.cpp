// Walks the dealing of the chunk attention's tiles (csrc/q36_chunk.h) on the host: what the workgroups run and write and
// what the combine reads, over many batches.  Prints each batch that fails and exits 1.
//   chunk_check SEED BATCHES
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#define __host__
#define __device__
#define __forceinline__ inline
#include "q36_chunk.h"

using namespace q36;

struct Cut {
  int b, h, tile, last;
};

static const char* walk(const std::vector<ChunkReq>& req, int G) {
  const int B = (int)req.size();
  int64_t total = 0;
  std::vector<std::vector<std::vector<int>>> done(2 * B);  // [request, head][tile][step]
  std::vector<std::vector<int>> written(2 * B);            // outputs written: by the tile's workgroup or the combine
  for (int b = 0; b < B; ++b) {
    total += ck_weight(req[b]);
    int sum = 0;
    const int nt = ck_tiles(req[b].n);
    for (int i = 0; i < nt; ++i) {
      if (ck_before(req[b], i) != sum) return "a tile's place is not the weight before it";
      if (ck_tile_at(req[b], sum) != i || ck_tile_at(req[b], sum + ck_steps(req[b], i) * ck_cost(req[b].n) + kTileOvh - 1) != i)
        return "a place's tile is not found";
      sum += ck_steps(req[b], i) * ck_cost(req[b].n) + kTileOvh;
      if (i + 1 == nt && ck_keys(req[b], i) != std::max(0, req[b].nk)) return "the last tile does not see all keys";
    }
    if (nt && (ck_before(req[b], nt) != sum || 2 * sum != ck_weight(req[b]))) return "a request's weight is not its tiles'";
    for (int h = 0; h < 2; ++h) {
      done[2 * b + h].resize(nt);
      for (int i = 0; i < nt; ++i) done[2 * b + h][i].assign(ck_steps(req[b], i), 0);
      written[2 * b + h].assign(nt, 0);
    }
  }
  if (total >= kMostWeight) return "a line that is too long";
  const int len = ck_share_len((int)total, G), nsh = ck_shares((int)total, len);
  if (nsh > G) return "more shares than workgroups";
  std::vector<long> owner(2 * G, -1);
  std::vector<Cut> cut(G, Cut{-1, 0, 0, 0});
  for (int w = 0; w < nsh; ++w) {
    const int x0 = w * len, x1 = std::min((int)total, x0 + len);
    if (x1 <= x0 || (w + 1 == nsh && x1 != total)) return "a share is empty, or the shares are not the line";
    // as the kernel walks: the request that x0 lies in, its head and tile, then on
    int b = 0;
    int at = 0;
    while (at + ck_weight(req[b]) <= x0) at += ck_weight(req[b++]);
    int h = 0, tile = 0;
    int off = at;
    if (req[b].n > 0) {
      const int head = ck_weight(req[b]) / 2;
      h = x0 - at >= head;
      off += h * head;
      tile = ck_tile_at(req[b], x0 - off);
      off += ck_before(req[b], tile);
    }
    while (off < x1) {
      if (req[b].n == 0) {
        ++off;
      } else {
        const int steps = ck_steps(req[b], tile), cost = ck_cost(req[b].n);
        const ChunkRun r = ck_run(steps, cost, off, x0, x1);
        if (r.nst >= 0) {
          if (r.st0 < 0 || r.st0 + r.nst > steps) return "a run outside its tile";
          for (int s = r.st0; s < r.st0 + r.nst; ++s) ++done[2 * b + h][tile][s];
          if (r.first && r.last) {
            ++written[2 * b + h][tile];
          } else {
            const int slot = ck_slot(w, r.first);
            if (owner[slot] >= 0) return "a slot written twice";
            owner[slot] = ((long)(2 * b + h) << 32) + tile;
            if (ck_first_share(steps, cost, off, len) != (r.first ? w : ck_first_share(steps, cost, off, len)) || (!r.first && ck_first_share(steps, cost, off, len) >= w))
              return "a tile's first share is not where it starts";
            if (r.first) cut[w] = Cut{b, h, tile, ck_last_share(steps, cost, off, len)};
          }
        }
        off += steps * cost + kTileOvh;
        if (++tile < ck_tiles(req[b].n)) continue;
        tile = 0;
        if (++h < 2) continue;
      }
      h = 0;
      if (++b >= B) break;
    }
  }
  int used = 0;
  for (int w = 0; w < G; ++w) {
    if (cut[w].b < 0) continue;
    const Cut c = cut[w];
    if (c.last <= w || c.last >= nsh) return "a cut tile that ends where it starts";
    for (int s = w; s <= c.last; ++s) {
      const int slot = ck_slot(s, s == w);
      if (owner[slot] != ((long)(2 * c.b + c.h) << 32) + c.tile) return "the combine reads a slot that this call did not write";
      ++used;
    }
    ++written[2 * c.b + c.h][c.tile];
  }
  if (used != (int)std::count_if(owner.begin(), owner.end(), [](long o) { return o >= 0; })) return "a partial not read";
  for (auto& t : done)
    for (auto& s : t)
      for (int d : s)
        if (d != 1) return "a step not in exactly one run";
  for (auto& t : written)
    for (int n : t)
      if (n != 1) return "a tile not written once";
  return nullptr;
}

int main(int argc, char** argv) {
  std::mt19937 g(argc > 1 ? atoi(argv[1]) : 0);
  const int batches = argc > 2 ? atoi(argv[2]) : 1000;
  auto uni = [&](int lo, int hi) { return (int)(lo + g() % (unsigned)(hi - lo + 1)); };
  auto logu = [&](int lo, int hi) {
    const double u = (double)g() / 4294967296.0;
    return std::max(lo, std::min(hi, (int)(lo * std::pow((hi + 1.0) / lo, u))));
  };
  int bad = 0;
  for (int a : {0, 1, 5, 1 << 29, kMostWeight - 1, kMostWeight})  // weights' sums stay between 0 and kMostWeight
    for (int b : {0, 1, 1 << 29, kMostWeight - 1, kMostWeight})
      if (ck_held(a, b) != (int)std::min<int64_t>((int64_t)a + b, kMostWeight)) printf("held(%d, %d) = %d\n", a, b, ck_held(a, b)), ++bad;
  auto check = [&](const std::vector<ChunkReq>& r, int G) {
    const char* e = walk(r, G);
    if (!e) return;
    if (++bad <= 10) {
      printf("B=%zu G=%d: %s:", r.size(), G, e);
      for (size_t i = 0; i < std::min<size_t>(r.size(), 6); ++i) printf(" (%d, %d)", r[i].n, r[i].nk);
      printf("\n");
    }
  };
  for (int n = 0; n <= 140; ++n)
    for (int nk : {0, 1, n / 2, n, n + 1, n + 31, n + 32, n + 63, n + 64, n + 500, n + 40000})
      for (int G : {1, 7, 256}) check({{n, nk}}, G);
  for (int i = 0; i < batches; ++i) {
    const int B = uni(0, 2) ? logu(1, 40) : logu(1, 900), hi = logu(1, B > 40 ? 300 : 9000), keys = logu(1, 40000);
    std::vector<ChunkReq> r(B);
    for (auto& q : r) {
      q.n = uni(0, 7) ? logu(1, hi) : uni(0, 1);
      q.nk = uni(0, 15) ? q.n + uni(0, keys) : uni(0, q.n);
    }
    check(r, uni(0, 7) ? 256 : uni(1, 304));
  }
  printf("%d of the batches fail\n", bad);
  return bad != 0;
}
