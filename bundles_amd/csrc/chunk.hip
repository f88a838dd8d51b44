// Attention of prompt chunks for gfx950 over the paged e4m3 KV cache: each request's new tokens (one to thousands) against
// all its keys, causal among the new ones, 16 query heads grouped onto 2 KV heads of 256 dims.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp2(s_j - m),  s_j = log2(e) scale (q . k_j),  m = max_j s_j
//
// (The reference re-pages the cache into 128-row pages and calls a library there, L/attn_fused.py:127-210.)
//
// Rounded: q to e4m3 (as attn_decode takes it), the weights p_j to f16 for the product with v (v is e4m3, exact in f16;
// 2^-11 a weight, where e4m3 weights would lose 2^-4; weights below 2^-21 of the row's largest by 2^-32 of it: kHead), the
// outputs to bf16.  Scores, maxima, weight sums and outputs: fp32.
//
// Bounds.  Long chunks: the matrix units, half the products at the e4m3 rate and half at the f16 one: 289 us for 8192 tokens
// from an empty cache at the rates of large library products (3161 and 1359 TFLOP/s); 389 to 425 measured (cards differ under
// this load), 1.29 to 1.41 PFLOP/s.  A step of 32 keys takes a workgroup 1.4 to 1.6 us (2.8 K cycles), of which the matrix
// units are busy 1.54 K and the vector units (scores to weights: 16 exponentials, maxima and sums a lane, and the values'
// widening, for 2 waves a SIMD) 1.6 K; the next block's scores formed beside this one's weights would overlap them better,
// and did not fit the registers (54 spilled).
// Short calls: the latency of one pass: lengths, shares and page tables 5 us, queries 2 to 5, a tile's end 3, the second
// launch 4: 17 us for five tokens over 300 keys.  Between: cut tiles, 256 KB a partial out of and back into the Infinity
// Cache (7 TB/s over the chip).
//
// Why so.  256 rows a workgroup: one pass over a tile's keys feeds eight waves from LDS (a wave alone would need four times
// the L2 rate).  LDS filled by copies past the registers: o holds 128 of a lane's 256 and q 32.  V^T by the transposing LDS
// read, P^T in the registers that S^T left it in: no shuffle between the products.  The running maximum lazily: o is scaled
// in the rare step in which a row has grown past 2^8 times (kLazyC).  Equal shares of one line: a call of any mix of lengths
// ends everywhere at once.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "q36_device.h"
#include "q36_host.h"
#include "q36_chunk.h"

namespace q36 {
namespace {

constexpr int kCHQ = 16, kCHKV = 2, kCD = 256, kCG = kCHQ / kCHKV;
constexpr int kCST = 32;  // keys a step

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef short v2s __attribute__((ext_vector_type(2)));
typedef unsigned short v2us __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));

struct ChunkDev {
  int B, T, sh, pt_stride, q8;
  int64_t num_slots;
  const void* q;
  const uint8_t* kc;
  const uint8_t* vc;
  const int32_t* pt;
  const int32_t* seqlens;
  const int32_t* qsl;
  uint16_t* out;
  float scale_log2;
  float* ws_o;   // [2 groups][8][8][4][64][4]: partial outputs of 8 waves' 32 rows, unnormalised
  float* ws_ml;  // [2 groups][8][2][32]: what their weights are relative to (base 2) and the weights' sums
  int4* cuts;    // [groups] the tile that starts in each share and is cut: request (-1: none), 2 tile + head, last share; and
                 // whether a value on the causal border was NaN
  uint32_t* flags;  // [groups] said when a share has written the partial that ends the tile which the share before starts; 0
                    // between calls (the combine kernel clears them: no call meets what another has said)
};

// A request's first row, new tokens and keys, inside the buffers whatever qsl and seqlens hold.
struct Req {
  int t0;
  ChunkReq r;
};
__device__ __forceinline__ Req req_of(const ChunkDev& d, int b) {
  const int t0 = min(max(d.qsl[b], 0), d.T), t1 = min(max(d.qsl[b + 1], t0), d.T);
  const int64_t keys = (int64_t)d.pt_stride << d.sh;
  return Req{t0, {t1 - t0, (int)min((int64_t)max(d.seqlens[b], 0), keys)}};
}
__device__ __forceinline__ v8h widen8(int w0, int w1) {
  const v2h a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.f, false);
  const v2h b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.f, true);
  const v2h c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.f, false);
  const v2h e = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.f, true);
  return v8h{a.x, a.y, b.x, b.y, c.x, c.y, e.x, e.y};
}
__device__ __forceinline__ v16f mfma_qk(v8i a, v8i b, v16f c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, 127, 0, 127);
}

// e4m3 NaN codes (0x7f, 0xff) of 4 bytes: bit 7 of each byte that is one.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// A step on the causal border multiplies some rows' values by a weight of zero, which would hand them a NaN that they do
// not see.  There the NaN values count as zero, and where a call has met one the combine kernel goes over the border's keys
// once more and puts the NaN where it is seen.

constexpr int kBlk = 2 * kCST * kCD;  // 32 keys in LDS: their K rows, then their V rows
constexpr int kSet = 4 * kBlk;
constexpr int kSlotF = 8 * 8 * 4 * 64 * 4, kSlotML = 8 * 2 * 32;  // floats of a partial
// Weights are relative to m, 7 binades below the row's maximum: the largest is 2^7, and the outputs are rescaled when the
// maximum has grown past 2^kLazyC times the one that m was taken from, so a weight is at most 2^15, inside f16.  f16 ends at
// half a step of 2^-25: 2^-32 of the largest weight, which 2^20 keys below it lose together as 2^-12 (with no head, 2^-5).
constexpr float kHead = 7.f;
// 8192 tokens at 0, 4, 8: 469, 438, 425 us; 2048 behind 6000 224, 209, 201.  (Past 8 a weight would leave f16.)
constexpr float kLazyC = 8.f;
// m lies a step of its own, 2^-23 |m| to 2^-22 |m|, below the maximum at the least, so that the maximum's weight is never lost
// to m's rounding.  Where scores can be so large that this step takes the room of f16 (256 products of 448^2 times the scale,
// past 2^23), weights are held at 2^(kHead + kLazyC): such rows' scores are equal to within their own rounding.
constexpr float kFarScale = 0x1p23f / (256.f * 448.f * 448.f);

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ void wait_vm0() { __builtin_amdgcn_s_waitcnt(0 | (7 << 4) | (15 << 8)); }
// 16 bytes a lane from memory into LDS at byte `at` + 16 lane of the workgroup's, past the registers.  In asm, so that the
// compiler does not hold each read of LDS back until every copy in flight has landed; the caller waits (wait_vm0).
__device__ __forceinline__ void copy16(const uint8_t* src, uint32_t at) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(at) : "memory");
}
__device__ __forceinline__ uint32_t lds_at(const void* p) {
  return (uint32_t)(uintptr_t)((const __attribute__((address_space(3))) uint8_t*)p);
}
__device__ __forceinline__ void barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// threadIdx.x through an empty asm: what is derived from it is formed afresh where it is used, in place of holding, or
// spilling, a register across the steps.
__device__ __forceinline__ int fresh_tid() {
  int t = (int)threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

__device__ __forceinline__ int wave_incl(int v) {  // inclusive sums over the wave, held at kMostWeight
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o);
    v = lane >= o ? ck_held(v, u) : v;
  }
  return v;
}

// A run of a tile's steps: what one workgroup does at a time.
struct Item {
  int b, t0, n, nk;   // the request: its number, first row, new tokens, keys
  int h, tok;         // KV head, the tile's first token
  int last;           // the last key that the tile's last token sees (0 where there is none)
  int key0, key1;     // the run's keys, key1 up to a step behind vis
  int slot;           // of its partial (-1: the whole tile)
  int lasts;          // of a tile's start: the share that has its end (-1: no start, or the whole tile)
  bool pair;          // the end of a tile that the share before starts
};

// The line of the call's tiles (q36_chunk.h), this workgroup's share of it, and its runs one after another, by 8 waves.
// Keys go by sets of four blocks of 32, between two barriers a set, out of one half of LDS while the other fills.  Wide tile:
// wave w has rows 32 w .. of the tile's 256 (4 tokens x 8 heads) and walks all the blocks.  Narrow: waves 2 k, 2 k + 1 have
// rows 0 .. 31, 32 .. 63 and walk block k of each set; the four are merged at the end.
// Scores S^T = K Q^T (32x32x64, e4m3): lane l holds row l % 32 and keys 8 (i / 4) + 4 (l / 32) + i % 4.  O^T += V^T P^T
// (32x32x16, f16): the lane's own weights in the order it has them, V^T by the transpose read from LDS rows in that order.
// A block of 32 keys in LDS: K row r holds key r, V row r key 16 (r / 16) + 8 ((r % 8) / 4) + 4 ((r / 8) % 2) + r % 4, 16-byte
// piece p of K row r at p ^ (r % 16), of V row r at p ^ 2 (r % 8): the 16 lanes' keys and the 32 lanes' values that are served
// together fall on all 16 of the row's bank slots.
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void chunk_kernel(ChunkDev d) {
  constexpr int NE = 4, SET = 32 * NE;  // a set's blocks, and a wave's copies of K and of V of one; its keys
  __shared__ __align__(1024) uint8_t X[2 * kSet];
  __shared__ float mlw[8][2][32];
  __shared__ int sums[8];
  __shared__ int found_at, found_b, nan_seen, joined;
  const int tid = threadIdx.x, wave = uni(tid >> 6), G = gridDim.x;
  // what a flag from this XCD says: not 0, and the XCD's number
  uint32_t xcc;
  asm("s_getreg_b32 %0, hwreg(HW_REG_XCC_ID)" : "=s"(xcc));
  const uint32_t mark = 16u | (xcc & 15u);
  // ---- this workgroup's share
  int total = 0, mine = 0;
  for (int c0 = 0; c0 < d.B; c0 += 512) {
    const int w = c0 + tid < d.B ? ck_weight(req_of(d, c0 + tid).r) : 0;
    mine = c0 ? ck_held(mine, w) : w;
  }
  if (tid == 0) nan_seen = 0;
  int inc = wave_incl(mine);
  if ((tid & 63) == 63) sums[wave] = inc;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    before = w == wave ? total : before;
    total = ck_held(total, sums[w]);
  }
  total = uni(total);
  const int len = ck_share_len(total, G), nsh = total < kMostWeight ? ck_shares(total, len) : 0;
  // neighbouring shares on one XCD (workgroup i runs on XCD i % 8): they walk the same keys, out of its L2
  const int xcd = blockIdx.x & 7, at8 = blockIdx.x >> 3, first = xcd * nsh / 8, count = (xcd + 1) * nsh / 8 - first;
  const int share = G % 8 ? (int)blockIdx.x : at8 < count ? first + at8 : nsh + (xcd * (G / 8) + at8) - (first + count);
  if (share >= nsh) {
    if (tid == 0 && share < G) d.cuts[share] = int4{-1, 0, 0, 0};
    return;
  }
  const int x0 = share * len, x1 = min(total, x0 + len);
  const bool joins = len >= kJoinShare;
  // the request that x0 lies in
  if (d.B <= 512) {
    const int off = before + inc - mine;
    if (off <= x0 && x0 < off + mine) found_b = tid, found_at = off;
    __syncthreads();
  } else {
    for (int c0 = 0, base = 0; base <= x0; c0 += 512) {
      const int w = c0 + tid < d.B ? ck_weight(req_of(d, c0 + tid).r) : 0;
      inc = wave_incl(w);
      __syncthreads();
      if ((tid & 63) == 63) sums[wave] = inc;
      __syncthreads();
      int off = base + inc - w;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        off += k < wave ? sums[k] : 0;
        base += sums[k];
      }
      if (off <= x0 && x0 < off + w) found_b = c0 + tid, found_at = off;
    }
    __syncthreads();
  }
  // the place on the line: request, head, tile
  int cb = 0, ct0 = 0, ch = 0, ctile = 0, coff = uni(found_at);
  ChunkReq cr = {0, 0};
  int4 cut = {-1, 0, 0, 0};
  auto request = [&](int b) {
    const Req q = req_of(d, b);
    cb = b, ct0 = uni(q.t0), cr = ChunkReq{uni(q.r.n), uni(q.r.nk)}, ch = 0, ctile = 0;
  };
  request(uni(found_b));
  if (cr.n > 0) {
    const int w = ck_weight(cr) >> 1;
    ch = x0 - coff >= w;
    coff += ch * w;
    ctile = ck_tile_at(cr, x0 - coff);
    coff += ck_before(cr, ctile);
  }
  // the share's next run (none: n = 0)
  auto next = [&] {
    Item it = {0, 0, 0, 0, 0, 0, 0, 0, 0, -1, -1, false};
    while (coff < x1 && it.n == 0) {
      if (cr.n == 0) {
        ++coff;
        if (coff < x1) request(cb + 1);
        continue;
      }
      const int steps = ck_steps(cr, ctile), ks = ck_step_keys(cr.n), cost = ck_cost(cr.n);
      const ChunkRun run = ck_run(steps, cost, coff, x0, x1);
      if (run.nst >= 0) {
        const bool whole = run.first && run.last;
        it = Item{cb, ct0, cr.n, cr.nk, ch, ctile * kWideTok, max(ck_keys(cr, ctile) - 1, 0), run.st0 * ks, (run.st0 + run.nst) * ks,
                  whole ? -1 : ck_slot(share, run.first), run.first && !whole ? ck_last_share(steps, cost, coff, len) : -1,
                  run.last && !whole && ck_first_share(steps, cost, coff, len) == share - 1};
      }
      coff += steps * cost + kTileOvh;
      if (++ctile < ck_tiles(cr.n)) continue;
      ctile = 0;
      if (++ch == 2 && coff < x1) request(cb + 1);
    }
    // scalars: what is made from them stays in SGPRs
    return Item{uni(it.b), uni(it.t0), uni(it.n), uni(it.nk), uni(it.h), uni(it.tok), uni(it.last), uni(it.key0), uni(it.key1), uni(it.slot), uni(it.lasts),
                uni(it.pair) != 0};
  };
  // ---- copies: wave w takes rows 4 w .. of each block's value rows and the same keys' rows; a lane has 16 bytes of row
  // `lane / 16` of the four
  const int top = (int)d.num_slots - 1, top_page = top >> d.sh, mask = (1 << d.sh) - 1;
  const int kap = 16 * (wave >> 2) + 8 * (wave & 1) + 4 * ((wave >> 1) & 1);  // the wave's first key of a block
  struct Ent {
    uint32_t v[NE];
  };
  // a set of keys: of request b, KV head h, from key0 on; behind key `last` this one again
  struct Keys {
    int b, h, key0, last;
  };
  auto keys_of = [](const Item& it, int set) { return Keys{it.b, it.h, it.key0 + set * SET, it.last}; };
  auto entries = [&](const Keys& k) {
    const int key = k.key0 + kap + ((fresh_tid() & 63) >> 4);
    const char* const pt = reinterpret_cast<const char*>(d.pt + (size_t)k.b * d.pt_stride);
    Ent x;
#pragma unroll
    for (int e = 0; e < NE; ++e) x.v[e] = *reinterpret_cast<const uint32_t*>(pt + (uint32_t)(min(key + 32 * e, k.last) >> d.sh) * 4u);
    return x;
  };
  auto copy = [&](const Keys& k, const Ent& x, int half) {
    const int lane = fresh_tid() & 63, t4 = lane >> 4, key = k.key0 + kap + t4;
    const uint8_t* const kbase = d.kc + (k.h * kCD + 16 * ((lane & 15) ^ ((kap & 15) + t4)));
    const uint8_t* const vbase = d.vc + (k.h * kCD + 16 * ((lane & 15) ^ (2 * (4 * (wave & 1) + t4))));
    const uint32_t to = (uint32_t)uni((int)lds_at(X) + half * kSet);
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const uint32_t pg = min(x.v[e], (uint32_t)top_page);  // (a negative number is a large one)
      const uint32_t sl = min((pg << d.sh) + (uint32_t)(min(key + 32 * e, k.last) & mask), (uint32_t)top);
      const uint64_t at = (uint64_t)sl << 9;
      copy16(kbase + at, to + e * kBlk + kap * kCD);
      copy16(vbase + at, to + e * kBlk + kCST * kCD + 4 * wave * kCD);
    }
  };
  // ---- the wave's rows of an item
  v8i qf[4];  // query fragments: column l % 32, dims 64 kb + 32 (l / 32) .. +31; rows of no token are zero
  v16f o[8];
  float m = 0.f, l = 0.f;
  int lim = -1;  // the row's last key
  uint32_t bad = 0;  // bits of NaN values on the causal border
  auto first_tok = [&](const Item& it) { return it.tok + 4 * (ck_wide(it.n) ? wave : wave & 1); };
  // this lane's places in a block: K row l % 32, piece 2 (l / 32) (the others: 4 kb + e more, by an xor); V row
  // 8 (l / 32) + (l % 16) / 2 (+ 16 c), piece (l / 16) % 2 (the others: 2 dt more)
  const int lane0 = tid & 63, g0 = lane0 >> 5;
  const uint32_t ka = (lane0 & 31) * kCD + 16 * ((2 * g0) ^ (lane0 & 15));
  const uint32_t va = kCST * kCD + (8 * g0 + ((lane0 & 15) >> 1)) * kCD + 16 * (((lane0 >> 4) & 1) ^ (lane0 & 14)) + 8 * (lane0 & 1);
  auto value = [&](uint32_t v0, int dt, int cc) {
    return __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)(uintptr_t)((v0 ^ (32 * dt)) + 16 * kCD * cc));
  };
  auto key = [&](uint32_t k0, int i) { return *(__attribute__((address_space(3))) const v4i*)(uintptr_t)(k0 ^ (16 * i)); };
  // The wave's query rows: read as they lie, 1 KB a load (four rows of codes, two of bf16), and handed out to the lanes
  // through the wave's 8 KB of `mem` (16-byte piece p of row r at p ^ (r % 16), as a block's keys).
  auto queries = [&](auto is_q8, const Item& it, uint8_t* mem) {
    constexpr bool q8 = decltype(is_q8)::value;
    const int lane = fresh_tid() & 63, tok = first_tok(it);
    const char* const rows = static_cast<const char*>(d.q) + (((size_t)(it.t0 + tok) * kCHQ + it.h * kCG) * kCD << (q8 ? 0 : 1));
    uint8_t* const my = mem + wave * 8192;
    v4i raw[q8 ? 8 : 16];
#pragma unroll
    for (int j = 0; j < (q8 ? 8 : 16); ++j) {
      const int r = q8 ? 4 * j + (lane >> 4) : 2 * j + (lane >> 5), at = q8 ? 256 * (r & 7) + 16 * (lane & 15) : 512 * (r & 7) + 16 * (lane & 31);
      raw[j] = v4i{0, 0, 0, 0};
      if (tok + (r >> 3) < it.n) raw[j] = *reinterpret_cast<const v4i*>(rows + (((size_t)(r >> 3) * kCHQ * kCD) << (q8 ? 0 : 1)) + at);
    }
    wait_vm0();  // (and the first item's first set of keys)
    if constexpr (q8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = 4 * j + (lane >> 4);
        *reinterpret_cast<v4i*>(my + 256 * r + 16 * ((lane & 15) ^ (r & 15))) = raw[j];
      }
    } else {
      // the conversion makes a NaN of what is past 448 (of 464, with its rounding): rows with one of those go the long way
      v2us big = {0, 0};
#pragma unroll
      for (int j = 0; j < 16; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) big = __builtin_elementwise_max(big, __builtin_bit_cast(v2us, raw[j][i] & 0x7fff7fff));
      }
      auto hand = [&](auto two) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int r = 2 * j + (lane >> 5);
          *reinterpret_cast<uint2*>(my + 256 * r + 16 * (((lane & 31) >> 1) ^ (r & 15)) + 8 * (lane & 1)) =
              make_uint2(two(raw[j].x, raw[j].y), two(raw[j].z, raw[j].w));
        }
      };
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(max(big.x, big.y) > 0x43e0) == 0, 1))
        hand([](int a, int b) {
          v2s r = {0, 0};
          r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(v2bf, a), 1.f, false);
          return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(v2bf, b), 1.f, true));
        });
      else
        hand([](int a, int b) {
          return f2e4m3x2_nan(bf_lo((uint32_t)a), bf_hi((uint32_t)a)) | (f2e4m3x2_nan(bf_lo((uint32_t)b), bf_hi((uint32_t)b)) << 16);
        });
    }
    const uint32_t k0 = lds_at(my) + ka;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      const v4i a = key(k0, 4 * kb), e = key(k0, 4 * kb + 1);
      qf[kb] = v8i{a.x, a.y, a.z, a.w, e.x, e.y, e.z, e.w};
    }
  };
  const float sl2 = d.scale_log2;
  const bool far = sl2 > kFarScale;
  bool begun = false;  // a block has been taken: m is of its rows' largest, and grows
  auto clean = [&](v2i w) {
    const uint32_t n0 = nan_bytes(w.x), n1 = nan_bytes(w.y);
    bad |= n0 | n1;
    return v2i{(int)(w.x & ~(n0 | (n0 - (n0 >> 7)))), (int)(w.y & ~(n1 | (n1 - (n1 >> 7))))};
  };
  // the block at byte `at` of LDS, keys key0 ..; border: some row does not see all of them
  auto block = [&](uint32_t at, int key0, bool border) {
    uint32_t k0 = at + ka, v0 = at + va;
    asm volatile("" : "+v"(k0), "+v"(v0));  // (the xors below are formed here, not held across blocks)
    v16f s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      const v4i a = key(k0, 4 * kb), e = key(k0, 4 * kb + 1);
      s = mfma_qk(v8i{a.x, a.y, a.z, a.w, e.x, e.y, e.z, e.w}, qf[kb], s);
    }
    v2i w[8];
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) w[dt] = value(v0, dt, 0);
    // (half of the keys' reads before the first product, the others and the values' between the products)
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
    if (border) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (key0 + 8 * (i >> 2) + 4 * g0 + (i & 3) > lim) s[i] = -INFINITY;
    }
    // relative to m, which the first block sets; where a row grows past 2^8 times the maximum that m is of, the row moves to
    // the new one.  (A row that sees nothing of a block sees nothing of the later ones.)
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; i += 2) mx = fmaxf(fmaxf(mx, s[i]), s[i + 1]);
    const auto p32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
    mx = fmaxf(__uint_as_float(p32[0]), __uint_as_float(p32[1]));
    const float top = __builtin_fmaf(mx, sl2, -m);
    if (__builtin_expect(!begun || __builtin_amdgcn_ballot_w64(top > kHead + kLazyC) != 0, 0)) {
      // (each row by its own maximum alone: its bits do not depend on its wave's other rows)
      const float x = mx * sl2, mn = top > (begun ? kHead + kLazyC : -INFINITY) ? x - fmaxf(kHead, fabsf(x) * 0x1p-23f) : m;
      const float al = begun ? __builtin_amdgcn_exp2f(m - mn) : 1.f;
      begun = true;
      m = mn;
      l *= al;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) o[dt] *= al;
    }
    // one formula for every block: equal scores get equal weights, however coarse m is at its size
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = __builtin_fmaf(s[i], sl2, -m);
    if (far) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = s[i] > kHead + kLazyC ? kHead + kLazyC : s[i];
    }
    v8h pb[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float p = __builtin_amdgcn_exp2f(s[i]);
      l += p;
      pb[i >> 3][i & 7] = (_Float16)p;
    }
    __builtin_amdgcn_sched_barrier(0);
    if (border) {
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) w[dt] = clean(w[dt]);
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(widen8(w[dt].x, w[dt].y), pb[0], o[dt], 0, 0, 0);
      w[dt] = value(v0, dt, 1);
    }
    if (border) {
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) w[dt] = clean(w[dt]);
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(widen8(w[dt].x, w[dt].y), pb[1], o[dt], 0, 0, 0);
  };
  // ---- the runs, one after another; while one ends, the first set of the next is on its way
  Item cur = {0, 0, 0, 0, 0, 0, 0, 0, 0, -1, -1, false}, nxt = next();
  // the keys that are copied next, and their page-table entries
  Keys ahead = keys_of(nxt, 0);
  Ent ent = {};
  if (nxt.n > 0) {
    copy(ahead, entries(ahead), 0);
    ahead.key0 += SET;
    ent = entries(ahead);
  }
  for (int half = 0;;) {
    uint8_t* const mem = X + (half ^ 1) * kSet;
    if (cur.n > 0) {
      l += __shfl_xor(l, 32);
      if (l == 0.f) m = -1e30f;  // no key seen
      const bool wide = ck_wide(cur.n);
      int slot = cur.slot;
      const int tok0 = first_tok(cur), rw = wide ? wave : wave & 1;
      const int lane = fresh_tid() & 63, col = lane & 31, g = lane >> 5;
      // A wide tile that the next share ends, most likely long ago, with its first run: where that partial is there, in this
      // XCD's L2, the two are joined here, by the combine kernel's arithmetic; else, and in calls of short shares
      // (kJoinShare), the combine kernel does it.
      // What makes this right without a release and an acquire, which would write back and empty whole caches: the flag says
      // the writer's XCD, so writer and reader share one L2; the writer waits until its stores have reached it before it says
      // so; the flag itself is read and written past the L1; and the reader's L1 has no line of the partial, since a launch
      // starts with an empty one and within a launch a partial is read once, here.  A second reader of a slot in the same
      // launch, on this CU, could meet an old line.
      bool join = false;
      if (joins && wide && cur.lasts == share + 1) {
        if (tid == 0) joined = __hip_atomic_load(d.flags + share + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == mark;
        barrier();
        join = uni(joined) != 0;
      }
      if (join) slot = -1;
      else if (cur.lasts >= 0) cut = int4{cur.b, 2 * (cur.tok / kWideTok) + cur.h, cur.lasts, 0};
      float* const wo = d.ws_o + (size_t)(slot < 0 ? 0 : slot) * kSlotF + (size_t)rw * (8 * 4 * 256) + lane * 4;
      float* const wml = d.ws_ml + (size_t)(slot < 0 ? 0 : slot) * kSlotML + rw * 64 + col;
      uint16_t* const rows = d.out + ((size_t)(cur.t0 + tok0) * kCHQ + cur.h * kCG) * kCD;  // row r: token r / 8, head r % 8
      if (!wide) {
        if (g == 0) mlw[wave][0][col] = m, mlw[wave][1][col] = l;
        barrier();
        float M = -1e30f, L = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) M = fmaxf(M, mlw[2 * k + rw][0][col]);
#pragma unroll
        for (int k = 0; k < 4; ++k) L += __builtin_amdgcn_exp2f(mlw[2 * k + rw][0][col] - M) * mlw[2 * k + rw][1][col];
        const float f = __builtin_amdgcn_exp2f(m - M), il = L > 0.f ? 1.f / L : L;
        if (slot >= 0 && wave < 2 && g == 0) wml[0] = M, wml[32] = L;
        // two dim tiles at a time through LDS, [wave][dt][a][lane]; wave (k, rw) sums quads 2 k, 2 k + 1 of the eight of rw
        // (rows 32 .. 63 only where there are more than 4 tokens: 4 requests of one token over 32000 keys 40.5 -> 39.5 us)
        const bool some = tok0 < cur.n;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (q) barrier();
          if (some) {
#pragma unroll
            for (int dt = 0; dt < 2; ++dt)
#pragma unroll
              for (int a = 0; a < 4; ++a)
                *reinterpret_cast<v4f*>(mem + wave * 8192 + (dt * 4 + a) * 1024 + lane * 16) =
                    v4f{o[2 * q + dt][4 * a] * f, o[2 * q + dt][4 * a + 1] * f, o[2 * q + dt][4 * a + 2] * f, o[2 * q + dt][4 * a + 3] * f};
          }
          barrier();
          if (some) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int quad = 2 * (wave >> 1) + u;
              v4f v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int k = 0; k < 4; ++k) v += *reinterpret_cast<const v4f*>(mem + (2 * k + rw) * 8192 + quad * 1024 + lane * 16);
              if (slot >= 0)
                *reinterpret_cast<v4f*>(wo + (8 * q + quad) * 256) = v;
              else if (tok0 + (col >> 3) < cur.n)
                *reinterpret_cast<uint2*>(rows + ((size_t)(col >> 3) * kCHQ + (col & 7)) * kCD + 64 * q + 8 * quad + 4 * g) =
                    make_uint2(pack_bf2_hw(v[0] * il, v[1] * il), pack_bf2_hw(v[2] * il, v[3] * il));
            }
          }
        }
      } else if (tok0 < cur.n) {
        if (slot < 0) {
          // rounded, through the wave's 8 KB of LDS (32 rows x 128 dims, 16-byte piece p of row r at p ^ (r % 16)), out by rows
          auto leave = [&](auto joins) {
            const float *o2 = nullptr;
            float f = 1.f, f2 = 0.f, L = l;
            if constexpr (decltype(joins)::value) {
              const size_t s2 = (size_t)ck_slot(share + 1, false);
              const float* const ml2 = d.ws_ml + s2 * kSlotML + wave * 64 + col;
              const float m2 = ml2[0], M = fmaxf(fmaxf(-1e30f, m), m2);
              o2 = d.ws_o + s2 * kSlotF + (size_t)wave * (8 * 4 * 256) + lane * 4;
              f = __builtin_amdgcn_exp2f(m - M), f2 = __builtin_amdgcn_exp2f(m2 - M);
              L = f * l + f2 * ml2[32];
            }
            const float il = L > 0.f ? 1.f / L : L;  // (no key: 0; NaN stays)
            uint8_t* const my = mem + wave * 8192;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
#pragma unroll
              for (int dt = 0; dt < 4; ++dt) {
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                  const v16f& u = o[4 * q + dt];
                  v4f v = {u[4 * a], u[4 * a + 1], u[4 * a + 2], u[4 * a + 3]};
                  if constexpr (decltype(joins)::value) v = f * v + f2 * *reinterpret_cast<const v4f*>(o2 + ((4 * q + dt) * 4 + a) * 256);
                  *reinterpret_cast<uint2*>(my + col * 256 + 16 * ((4 * dt + a) ^ (col & 15)) + 8 * g) =
                      make_uint2(pack_bf2_hw(v[0] * il, v[1] * il), pack_bf2_hw(v[2] * il, v[3] * il));
                }
                if (decltype(joins)::value && (dt & 1)) __builtin_amdgcn_sched_barrier(0);  // (eight loads in flight, no more registers)
              }
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const int row = 4 * j + (lane >> 4);
                const v4i v = *reinterpret_cast<const v4i*>(my + row * 256 + 16 * ((lane & 15) ^ (row & 15)));
                if (tok0 + (row >> 3) < cur.n)
                  __builtin_nontemporal_store(v, reinterpret_cast<v4i*>(rows + ((size_t)(row >> 3) * kCHQ + (row & 7)) * kCD + 128 * q + 8 * (lane & 15)));
              }
            }
          };
          join ? leave(std::true_type{}) : leave(std::false_type{});
        } else {
#pragma unroll
          for (int dt = 0; dt < 8; ++dt)
#pragma unroll
            for (int a = 0; a < 4; ++a)
              *reinterpret_cast<v4f*>(wo + (dt * 4 + a) * 256) = v4f{o[dt][4 * a], o[dt][4 * a + 1], o[dt][4 * a + 2], o[dt][4 * a + 3]};
          if (g == 0) wml[0] = m, wml[32] = l;
        }
      }
      if (joins && wide && cur.pair) {
        wait_vm0();
        barrier();  // the partial is in L2
        if (tid == 0) __hip_atomic_store(d.flags + share, mark, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      if (!wide) barrier();  // (the waves' LDS is theirs again)
    }
    if (nxt.n == 0) break;
    d.q8 ? queries(std::true_type{}, nxt, mem) : queries(std::false_type{}, nxt, mem);
    cur = nxt;
    nxt = next();
    const bool wide = ck_wide(cur.n);
    const int sets = max(1, (cur.key1 - cur.key0 + SET - 1) / SET), tok0 = first_tok(cur), pre = cur.nk - cur.n;
    if (sets == 1) ahead = keys_of(nxt, 0), ent = entries(ahead);  // (those on their way are behind this item's end)
    {
      const int tok = tok0 + ((fresh_tid() & 31) >> 3);
      lim = tok < cur.n ? pre + tok : -1;
      m = 0.f, l = 0.f;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
    }
    begun = false;
    // the wave's keys: of the run, up to its last token's; none without a token
    const int end = uni(tok0 < cur.n ? min(pre + min(tok0 + 4, cur.n), cur.key1) : 0);
#pragma unroll 1
    for (int st = 0; st < sets; ++st) {
      wait_vm0();  // (also said of an item's first set, so that no wait for the entries stands among the copies)
      barrier();  // every wave's copies of this set have landed, and every wave is done with the other half
      // the next set, this item's or the next one's, and the page-table entries of the one behind it
      if (st + 1 < sets || nxt.n > 0) {
        copy(ahead, ent, half ^ 1);
        ahead.key0 += SET;
        if (st + 2 == sets) ahead = keys_of(nxt, 0);
        ahead = Keys{uni(ahead.b), uni(ahead.h), uni(ahead.key0), uni(ahead.last)};
        ent = entries(ahead);
      }
      const uint32_t to = lds_at(X) + half * kSet;
      const int i1 = wide ? NE : (wave >> 1) + 1;
#pragma unroll 1
      for (int i = wide ? 0 : wave >> 1; i < i1; ++i) {
        const int k = cur.key0 + st * SET + 32 * i;
        if (k >= end) break;
        // a SIMD's older wave wins where both could issue, and its other one would then end each set alone: they take turns
        // (8192 tokens 434 -> 425 us, 2048 behind 6000 207 -> 201)
        if (((i >> 1) ^ (wave >> 2)) & 1) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
        block(to + i * kBlk, k, k + 31 > pre + tok0);
      }
      half ^= 1;
    }
    wait_vm0();
    barrier();  // every wave is done with this item's last set (the other half than `half`), and the next item's first has landed
  }
  if (__builtin_amdgcn_ballot_w64(bad != 0) && (tid & 63) == 0) nan_seen = 1;
  __syncthreads();
  if (tid == 0) {
    cut.w = nan_seen;
    d.cuts[share] = cut;
  }
}

// Which of the values at dims dim .. dim + 3 (bit 7 of each byte) are NaN at a key on the border that new token tok sees.
__device__ __forceinline__ uint32_t border_nans(const ChunkDev& d, int b, ChunkReq r, int h, int tok, int dim) {
  const int pre = r.nk - r.n;
  uint32_t n = 0;
  for (int key = max(0, pre + (tok & ~3) - 31); key <= pre + tok; ++key) {
    const int top = (int)d.num_slots - 1, pg = min(max(d.pt[(size_t)b * d.pt_stride + (key >> d.sh)], 0), top >> d.sh);
    const int sl = min((pg << d.sh) + (key & ((1 << d.sh) - 1)), top);
    n |= nan_bytes(*reinterpret_cast<const uint32_t*>(d.vc + ((size_t)sl * kCHKV + h) * kCD + dim));
  }
  return n;
}
__device__ __forceinline__ uint2 put_nans(uint2 v, uint32_t n) {
  const uint32_t q = 0x7fc0;
  return make_uint2((n & 0x80 ? (v.x & 0xffff0000u) | q : v.x) | (n & 0x8000 ? 0xffff0000u : 0), (n & 0x800000 ? (v.y & 0xffff0000u) | q : v.y) | (n & 0x80000000u ? 0xffff0000u : 0));
}

// The cut tiles: out = bf16(sum_p exp2(m_p - M) o_p / sum_p exp2(m_p - M) l_p) over a tile's partials p.  Up to kFew partials:
// a workgroup takes 32 rows and 64 dims at a time, wave a the lanes' a-th four dims of each 32, four partials' loads in
// flight.  More: 32 rows and 8 dims, wave w has partials w, w + 4, .., eight at a time, and the waves' sums meet in LDS: four
// times the workgroups for a tile, for tiles that are few.  Bound by the partials' bytes, out of the Infinity Cache: 2048
// tokens behind 6000 (128 tiles, 3 partials each, 96 MB) in 20 us.  us a call at kFew 4, 16, 32, 256: three chunks of 130 ..
// 300 tokens over long contexts (6 partials a tile) 243, 232, 232, 233; two of 90 tokens behind 30000 (21) 95, 95, 92, 92; one
// of 32 behind 32000 (128) 46, 46, 46, 58.
constexpr int kFew = 32;
__global__ __launch_bounds__(256) void chunk_combine_kernel(ChunkDev d, int G) {
  // request and partials (16 bits each), 2 tile + head (20 bits) and share: few partials from the front, many from the back
  __shared__ uint2 list[1024];
  __shared__ int counts[4][2], nan_flags[4];
  __shared__ v4f part[4][64];
  __shared__ float pml[4][2][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), col = lane & 31, g = lane >> 5;
  // the shares that leave a cut tile, in order
  int few = 0, many = 0;
  uint64_t nans = 0;
  for (int c0 = 0; c0 < G; c0 += 256) {
    const int4 c = c0 + tid < G ? d.cuts[c0 + tid] : int4{-1, 0, 0, 0};
    const int n = c.x >= 0 ? c.z - (c0 + tid) + 1 : 0;
    nans |= __builtin_amdgcn_ballot_w64(c.w != 0);
    const uint64_t fb = __builtin_amdgcn_ballot_w64(n > 0 && n <= kFew), mb = __builtin_amdgcn_ballot_w64(n > kFew), below = (1ull << lane) - 1;
    if (lane == 0) counts[wave][0] = __builtin_popcountll(fb), counts[wave][1] = __builtin_popcountll(mb);
    __syncthreads();
    int fat = few + __builtin_popcountll(fb & below), mat = many + __builtin_popcountll(mb & below);
    for (int w = 0; w < 4; ++w) {
      fat += w < wave ? counts[w][0] : 0, mat += w < wave ? counts[w][1] : 0;
      few += counts[w][0], many += counts[w][1];
    }
    if (n > 0) list[n <= kFew ? fat : 1023 - mat] = make_uint2((uint32_t)c.x << 16 | (uint32_t)n, (uint32_t)c.y << 12 | (uint32_t)(c0 + tid));
    __syncthreads();
  }
  if (blockIdx.x == 0)
    for (int i = tid; i < G; i += 256) __hip_atomic_store(d.flags + i, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (lane == 0) nan_flags[wave] = nans != 0;
  __syncthreads();
  const bool any_nan = uni(nan_flags[0] | nan_flags[1] | nan_flags[2] | nan_flags[3]) != 0;
  few = uni(few), many = uni(many);
  for (int unit = blockIdx.x; unit < few * 32 + many * 256; unit += gridDim.x) {
    const int mu = unit - few * 32;
    const uint2 c = list[mu < 0 ? unit >> 5 : 1023 - (mu >> 8)];
    const int rw = mu < 0 ? (unit >> 2) & 7 : (mu >> 5) & 7, b = uni((int)(c.x >> 16)), n = uni((int)(c.x & 0xffffu));
    const int tile = uni((int)(c.y >> 13)), h = uni((int)(c.y >> 12)) & 1, share = uni((int)(c.y & 0xfffu));
    const Req q = req_of(d, b);
    const int tok = tile * kWideTok + 4 * rw + (col >> 3), head = h * kCG + (col & 7);
    if ((!ck_wide(q.r.n) && rw >= 2) || uni(tok) >= q.r.n) continue;
    const bool row_ok = tok < q.r.n;
    // (bases in scalars, a lane's part a 32-bit offset)
    auto ml = [&](int p, int what) {
      const char* const at = reinterpret_cast<const char*>(d.ws_ml + (size_t)uni(ck_slot(share + p, p == 0)) * kSlotML + rw * 64 + 32 * what);
      return *reinterpret_cast<const float*>(at + (uint32_t)col * 4u);
    };
    auto po = [&](int p, int dt, int a) {
      const char* const at = reinterpret_cast<const char*>(d.ws_o + (size_t)uni(ck_slot(share + p, p == 0)) * kSlotF + ((rw * 8 + dt) * 4 + a) * 256);
      return *reinterpret_cast<const v4f*>(at + (uint32_t)lane * 16u);
    };
    auto store = [&](int dt, int a, v4f v, float L) {
      const float il = L > 0.f ? 1.f / L : L;
      const int dim = 32 * dt + 8 * a + 4 * g;
      uint2 w = make_uint2(pack_bf2_hw(v[0] * il, v[1] * il), pack_bf2_hw(v[2] * il, v[3] * il));
      if (__builtin_expect(any_nan, 0)) w = put_nans(w, border_nans(d, b, q.r, h, tok, dim));
      *reinterpret_cast<uint2*>(d.out + ((size_t)(q.t0 + tok) * kCHQ + head) * kCD + dim) = w;
    };
    if (mu < 0) {
      const int dt = 2 * (unit & 3);
      float M = -1e30f, L = 0.f;
      v4f s[2] = {};
#pragma unroll 1
      for (int p0 = 0; p0 < n; p0 += 4) {
        float mp[4], lp[4], mn = M;
        v4f v[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          mp[i] = -1e30f, lp[i] = 0.f;
          if (p0 + i < n) mp[i] = ml(p0 + i, 0), lp[i] = ml(p0 + i, 1), v[i][0] = po(p0 + i, dt, wave), v[i][1] = po(p0 + i, dt + 1, wave);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) mn = fmaxf(mn, mp[i]);
        const float f = __builtin_amdgcn_exp2f(M - mn);
        M = mn, L *= f, s[0] *= f, s[1] *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (p0 + i < n) {
            const float w = __builtin_amdgcn_exp2f(mp[i] - M);
            L += w * lp[i], s[0] += w * v[i][0], s[1] += w * v[i][1];
          }
        }
      }
      if (row_ok) store(dt, wave, s[0], L), store(dt + 1, wave, s[1], L);
      continue;
    }
    const int dt = (mu >> 2) & 7, a = mu & 3;
    float M = -1e30f, L = 0.f;
    v4f s = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = wave; p0 < n; p0 += 32) {
      float mp[8], lp[8], mn = M;
      v4f v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        mp[i] = -1e30f, lp[i] = 0.f;
        if (p0 + 4 * i < n) mp[i] = ml(p0 + 4 * i, 0), lp[i] = ml(p0 + 4 * i, 1), v[i] = po(p0 + 4 * i, dt, a);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) mn = fmaxf(mn, mp[i]);
      const float f = __builtin_amdgcn_exp2f(M - mn);
      M = mn, L *= f, s *= f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (p0 + 4 * i < n) {
          const float w = __builtin_amdgcn_exp2f(mp[i] - M);
          L += w * lp[i], s += w * v[i];
        }
      }
    }
    pml[wave][0][lane] = M, pml[wave][1][lane] = L;
    part[wave][lane] = s;
    __syncthreads();
    if (wave == 0) {
      const float Ma = fmaxf(fmaxf(pml[0][0][lane], pml[1][0][lane]), fmaxf(pml[2][0][lane], pml[3][0][lane]));
      float La = 0.f;
      v4f t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(pml[w][0][lane] - Ma);
        La += f * pml[w][1][lane];
        t += f * part[w][lane];
      }
      if (row_ok) store(dt, a, t, La);
    }
    __syncthreads();
  }
  if (__builtin_expect(!any_nan, 1)) return;
  // every new token and KV head, a thread 4 dims: the NaN that the tiles' own workgroups left out (a cut tile's are there)
  for (int b = 0; b < d.B; ++b) {
    const Req q = req_of(d, b);
    for (int64_t i = (int64_t)blockIdx.x * 256 + tid; i < (int64_t)q.r.n * (2 * kCD / 4); i += (int64_t)gridDim.x * 256) {
      const int tok = (int)(i / (2 * kCD / 4)), h = (int)(i / (kCD / 4)) & 1, dim = 4 * (int)(i % (kCD / 4));
      const uint32_t n = border_nans(d, b, q.r, h, tok, dim);
      if (n)
        for (int e = 0; e < 4; ++e)
          if (n >> (8 * e + 7) & 1)
            for (int hd = 0; hd < kCG; ++hd) d.out[((size_t)(q.t0 + tok) * kCHQ + h * kCG + hd) * kCD + dim + e] = 0x7fc0;
    }
  }
}

// A workspace before its first call: no partial said to be there.
__global__ __launch_bounds__(256) void chunk_init_kernel(uint32_t* flags, int G) {
  for (int i = threadIdx.x; i < G; i += 256) flags[i] = 0;
}

// Workgroups: one a CU (their LDS and registers fill it).
int chunk_groups() { return std::min(std::max(device_cus(), 1), 1024); }
struct ChunkWs {
  size_t o, ml, cuts, flags, total;
};
ChunkWs chunk_ws(int G) {
  ChunkWs w;
  w.o = 0;
  w.ml = align_up(w.o + sizeof(float) * 2 * (size_t)G * kSlotF, 256);
  w.cuts = align_up(w.ml + sizeof(float) * 2 * (size_t)G * kSlotML, 256);
  w.flags = align_up(w.cuts + sizeof(int4) * (size_t)G, 256);
  w.total = align_up(w.flags + sizeof(uint32_t) * (size_t)G, 256);
  return w;
}

}  // namespace
}  // namespace q36

using namespace q36;

extern "C" size_t q36_attn_chunk_workspace_bytes(void) { return chunk_ws(chunk_groups()).total; }

extern "C" int q36_attn_chunk_workspace_init(void* workspace, size_t workspace_bytes, q36_stream_t stream) {
  const int G = chunk_groups();
  const ChunkWs L = chunk_ws(G);
  Q36_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, "q36_attn_chunk_workspace_init: workspace must be 256-byte aligned");
  Q36_REQUIRE(workspace_bytes >= L.total, "q36_attn_chunk_workspace_init: workspace of %zu bytes < %zu required", workspace_bytes, L.total);
  chunk_init_kernel<<<1, 256, 0, static_cast<hipStream_t>(stream)>>>(reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + L.flags), G);
  return check_launch("q36_attn_chunk_workspace_init");
}

extern "C" int q36_attn_chunk(const q36_chunk_args* a, q36_stream_t stream) {
  Q36_REQUIRE(a != nullptr, "q36_attn_chunk: null args");
  Q36_REQUIRE(a->HQ == kCHQ && a->HKV == kCHKV && a->D == kCD, "q36_attn_chunk: HQ=%d HKV=%d D=%d unsupported (this build: 16 / 2 / 256)",
              a->HQ, a->HKV, a->D);
  Q36_REQUIRE(a->B >= 1 && a->B <= 65535 && a->T >= 1 && a->T <= (1 << 20), "q36_attn_chunk: B=%d T=%d out of range", a->B, a->T);
  Q36_REQUIRE(a->page_size >= 1 && a->page_size <= 1024 && (a->page_size & (a->page_size - 1)) == 0,
              "q36_attn_chunk: page_size=%d must be a power of two up to 1024", a->page_size);
  Q36_REQUIRE(a->pt_stride >= 1 && a->pt_stride <= (1 << 27) / a->page_size, "q36_attn_chunk: pt_stride=%d of pages of %d out of range",
              a->pt_stride, a->page_size);
  Q36_REQUIRE(!ck_too_long(a->T, a->B, (int64_t)a->pt_stride * a->page_size),
              "q36_attn_chunk: T=%d, B=%d with tables of %d pages of %d: more steps than one call deals", a->T, a->B, a->pt_stride,
              a->page_size);
  Q36_REQUIRE(a->num_slots >= 1 && a->num_slots < ((int64_t)1 << 31), "q36_attn_chunk: num_slots=%lld out of range",
              (long long)a->num_slots);
  Q36_REQUIRE(a->q && a->k_cache && a->v_cache && a->page_table && a->seqlens && a->qsl && a->out && a->workspace,
              "q36_attn_chunk: a required pointer is null");
  Q36_REQUIRE(aligned16(a->q) && aligned16(a->k_cache) && aligned16(a->v_cache) && aligned16(a->out) &&
                  (reinterpret_cast<uintptr_t>(a->workspace) & 255u) == 0,
              "q36_attn_chunk: q, out and the caches must be 16-byte and workspace 256-byte aligned");
  Q36_REQUIRE(a->scale > 0.f && a->scale <= 1e6f, "q36_attn_chunk: scale=%g out of range", (double)a->scale);
  const int G = chunk_groups();
  const ChunkWs L = chunk_ws(G);
  Q36_REQUIRE(a->workspace_bytes >= L.total, "q36_attn_chunk: workspace of %zu bytes < %zu required", a->workspace_bytes, L.total);
  int sh = 0;
  while ((1 << sh) < a->page_size) ++sh;
  char* const ws = static_cast<char*>(a->workspace);
  const ChunkDev d{a->B, a->T, sh, a->pt_stride, a->q_e4m3, a->num_slots, a->q, static_cast<const uint8_t*>(a->k_cache),
                   static_cast<const uint8_t*>(a->v_cache), a->page_table, a->seqlens, a->qsl, static_cast<uint16_t*>(a->out),
                   a->scale * 1.44269504088896340736f, reinterpret_cast<float*>(ws + L.o), reinterpret_cast<float*>(ws + L.ml),
                   reinterpret_cast<int4*>(ws + L.cuts), reinterpret_cast<uint32_t*>(ws + L.flags)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  chunk_kernel<<<G, 512, 0, st>>>(d);
  chunk_combine_kernel<<<1024, 256, 0, st>>>(d, G);
  return check_launch("q36_attn_chunk");
}
