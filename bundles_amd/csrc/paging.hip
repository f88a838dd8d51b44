// The page plan of a step: from the requests' cached and new token counts, the row starts, key counts, positions
// and cache slots of the new tokens, the block tables extended by pages of the free list, and (optionally) the
// one-token page table that decode attention reads.  (No reference counterpart: the reference takes out_cache_loc,
// page_table and cache_seqlens_int32 from its serving engine, L/attn_fused.py:70-75.)
//
//   qsl_b = sum_{a<b} new_a,  seqlens_b = cached_b + new_b,  have_b = ceil(cached_b / P)
//   need_b = ceil(seqlens_b / P) - have_b,  off_b = sum_{a<b} need_a
//   page(b, j) = j < have_b ? table[row_b][j] : free[off_b + j - have_b]
//   token i of request b: position cached_b + i, slot page(b, position / P) * P + position % P
//
// One launch: a workgroup takes a segment of one request and forms that request's two prefix sums from the counts of
// the requests before it (8 bytes a request, in L2), so no workgroup waits for another.  New pages are read from the
// free list, never from a table entry that another workgroup writes.  Bound by the launch and two loads behind one another
// (lengths, then pages): 3.9 us on the GPU for 7 decoding requests, 5.5 for 203 of up to 8191 keys (1.1 MB), 10.6 for 256 of
// up to 32000 (14 MB, 1.3 TB/s); a call from Python takes 8 us at the least.
#include <algorithm>

#include "q36_device.h"
#include "q36_host.h"
#include "q36_plan.h"

namespace q36 {
namespace {

struct PlanDev {
  int B, T, sh, rows, width, nfree, pt_width, whole, segs;
  const int32_t *cached, *fresh, *req;
  int32_t* table;
  const int32_t* free_pages;
  int32_t *qsl, *seqlens, *positions;
  int64_t* out_loc;
  int32_t *used, *page_table;
};

__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* sums) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
  __syncthreads();
  v = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  __syncthreads();
  return v;
}

__global__ __launch_bounds__(256) void page_plan_kernel(PlanDev d) {
  __shared__ int64_t sums[4];
  const int b = blockIdx.x / d.segs, seg = blockIdx.x % d.segs, tid = threadIdx.x, sh = d.sh, P = 1 << sh;
  const int cached = count_of(d.cached[b]), fresh = count_of(d.fresh[b]);
  const int row = d.req ? d.req[b] : b;
  const bool row_ok = row >= 0 && row < d.rows;
  int64_t first = 0, off = 0;  // tokens and new pages of the requests before this one
  for (int a = tid; a < b; a += 256) {
    const int c = count_of(d.cached[a]), n = count_of(d.fresh[a]);
    first += n;
    off += pages_of(c + n, sh) - pages_of(c, sh);
  }
  if (b > 0) {
    first = block_sum(first, sums);
    off = block_sum(off, sums);
  }
  const int len = cached + fresh, have = pages_of(cached, sh), full = pages_of(len, sh);
  int32_t* const tab = d.table + (size_t)(row_ok ? row : 0) * d.width;
  const int most = 0x7fffffff >> sh;  // page numbers whose slots fit 31 bits
  // page j of the request, -1 where there is none (past the table, past the free list, a number out of range)
  auto page_of = [&](int j) -> int {
    if (!row_ok || j >= d.width) return -1;
    int p = -1;
    if (j < have) p = tab[j];
    else if (off + (j - have) < d.nfree) p = d.free_pages[off + (j - have)];
    return p < 0 || p >= most ? -1 : p;
  };
  const int step = 256 * d.segs, at = 256 * seg + tid;
  // the new tokens
  const int64_t tokens = min((int64_t)fresh, max((int64_t)d.T - first, (int64_t)0));
  for (int i = at; i < tokens; i += step) {
    const int pos = cached + i, pg = page_of(pos >> sh);
    const bool ok = pg >= 0 && (!d.page_table || pos < d.pt_width);
    d.positions[first + i] = pos;
    d.out_loc[first + i] = ok ? (int64_t)pg * P + (pos & (P - 1)) : -1;
  }
  // the table's new pages
  if (row_ok)
    for (int j = have + at; j < min(full, d.width); j += step)
      if (off + (j - have) < d.nfree) tab[j] = d.free_pages[off + (j - have)];
  // the one-token page table: all keys or the new ones; a key without a page gets slot 0
  if (d.page_table) {
    int32_t* const pt = d.page_table + (size_t)b * d.pt_width;
    for (int i = (d.whole ? 0 : cached) + at; i < min(len, d.pt_width); i += step) {
      const int pg = page_of(i >> sh);
      pt[i] = pg >= 0 ? pg * P + (i & (P - 1)) : 0;
    }
  }
  if (seg == 0 && tid == 0) {
    d.qsl[b] = (int)min(first, (int64_t)d.T);
    d.seqlens[b] = len;
  }
  if (b == d.B - 1) {
    // rows behind the last request: position 0 and no slot, as a padded batch has them
    for (int64_t t = first + fresh + at; t < d.T; t += step) {
      d.positions[t] = 0;
      d.out_loc[t] = -1;
    }
    if (seg == 0) {
      // what did not fit, over all requests (the bits of the header)
      int bits = 0;
      for (int a = tid; a < d.B; a += 256) {
        const int c = count_of(d.cached[a]), n = count_of(d.fresh[a]), r = d.req ? d.req[a] : a;
        if (r < 0 || r >= d.rows || pages_of(c + n, sh) > d.width || c < d.cached[a] || n < d.fresh[a]) bits |= Q36_PLAN_TABLE;
        if (d.page_table && c + n > d.pt_width) bits |= Q36_PLAN_PAGE_TABLE;
      }
      const int64_t tokens_all = first + fresh, pages_all = off + (full - have);
      if (tokens_all > d.T) bits |= Q36_PLAN_TOKENS;
      if (pages_all > d.nfree) bits |= Q36_PLAN_PAGES;
      const uint64_t any0 = __builtin_amdgcn_ballot_w64(bits & 1), any1 = __builtin_amdgcn_ballot_w64(bits & 2),
                     any2 = __builtin_amdgcn_ballot_w64(bits & 4), any3 = __builtin_amdgcn_ballot_w64(bits & 8);
      if ((tid & 63) == 0) sums[tid >> 6] = (any0 ? 1 : 0) | (any1 ? 2 : 0) | (any2 ? 4 : 0) | (any3 ? 8 : 0);
      __syncthreads();
      if (tid == 0) {
        d.qsl[d.B] = (int)min(tokens_all, (int64_t)d.T);
        d.used[0] = (int)min(pages_all, (int64_t)d.nfree);
        d.used[1] = (int)(sums[0] | sums[1] | sums[2] | sums[3]);
      }
    }
  }
}

}  // namespace
}  // namespace q36

using namespace q36;

extern "C" int q36_page_plan(const q36_page_plan_args* a, q36_stream_t stream) {
  Q36_REQUIRE(a != nullptr, "q36_page_plan: null args");
  Q36_REQUIRE(a->B >= 1 && a->B <= 65535 && a->T >= 0, "q36_page_plan: B=%d T=%d out of range", a->B, a->T);
  Q36_REQUIRE(a->page_size >= 1 && a->page_size <= 1024 && (a->page_size & (a->page_size - 1)) == 0,
              "q36_page_plan: page_size=%d must be a power of two up to 1024", a->page_size);
  Q36_REQUIRE(a->table_rows >= 1 && a->table_width >= 1 && a->free_count >= 0,
              "q36_page_plan: table of %d x %d, %d free pages", a->table_rows, a->table_width, a->free_count);
  Q36_REQUIRE(a->req || a->table_rows >= a->B, "q36_page_plan: a table of %d rows for B=%d without req", a->table_rows, a->B);
  Q36_REQUIRE(a->cached && a->new_tokens && a->table && a->qsl && a->seqlens && a->used &&
                  (a->free_count == 0 || a->free_pages) && (a->T == 0 || (a->positions && a->out_loc)),
              "q36_page_plan: a required pointer is null");
  Q36_REQUIRE(!a->page_table || a->pt_width >= 1, "q36_page_plan: page table of width %d", a->pt_width);
  int sh = 0;
  while ((1 << sh) < a->page_size) ++sh;
  // Segments: 2048 keys or tokens a workgroup where the batch is small, no more workgroups than fill the chip's CUs eight
  // times over (a segment's threads walk on through a longer request).  On the GPU, at 512 / 2048 / 8192 keys a segment: 203
  // requests of up to 8191 keys 6.5 / 5.5 / 6.8 us, 256 of up to 32000 10.6 / 10.6 / 12.5.
  const int most = std::max(a->page_table && a->whole ? a->pt_width : 0, a->T / a->B);
  const int segs = std::max(1, std::min((most - 1) / 2048 + 1, std::max(1, 2048 / a->B)));
  PlanDev d{a->B, a->T, sh, a->table_rows, a->table_width, a->free_count, a->pt_width, a->whole ? 1 : 0, segs,
            a->cached, a->new_tokens, a->req, a->table, a->free_pages, a->qsl, a->seqlens, a->positions, a->out_loc,
            a->used, a->page_table};
  page_plan_kernel<<<(unsigned)a->B * segs, 256, 0, static_cast<hipStream_t>(stream)>>>(d);
  return check_launch("q36_page_plan");
}
