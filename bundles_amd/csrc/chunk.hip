// Attention of prompt chunks for gfx950 over the paged e4m3 KV cache: each request's new tokens (one to thousands) against
// all its keys, causal among the new ones, 16 query heads grouped onto 2 KV heads of 256 dims.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp2(s_j - m),  s_j = log2(e) scale (q . k_j),  m = max_j s_j
//
// (The reference re-pages the cache into 128-row pages and calls a library there, L/attn_fused.py:127-210.)
#include <math.h>

#include "q36_device.h"
#include "q36_host.h"

namespace q36 {
namespace {

constexpr int kCHQ = 16, kCHKV = 2, kCD = 256, kCG = kCHQ / kCHKV;
constexpr int kCST = 32;  // keys a step

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
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
};

// A request's new tokens and keys, inside the buffers whatever qsl and seqlens hold.
struct Req {
  int t0, n, nk;
};
__device__ __forceinline__ Req req_of(const ChunkDev& d, int b) {
  const int t0 = min(max(d.qsl[b], 0), d.T), t1 = min(max(d.qsl[b + 1], t0), d.T);
  const int64_t keys = (int64_t)d.pt_stride << d.sh;
  return Req{t0, t1 - t0, (int)min((int64_t)max(d.seqlens[b], 0), keys)};
}
__device__ __forceinline__ int64_t slot_of(const ChunkDev& d, int b, int key) {
  const int64_t p = d.pt[(size_t)b * d.pt_stride + (key >> d.sh)];
  const int64_t s = (p << d.sh) + (key & ((1 << d.sh) - 1));
  return s < 0 ? 0 : s >= d.num_slots ? d.num_slots - 1 : s;
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
// not see.  There the NaN values count as zero, and a product of two indicators (value is NaN, key is seen) finds the
// outputs that do see one.
//
// One wave: 4 new tokens x 8 query heads (32 rows) of a KV head over all their keys, 32 keys a step.
// Scores S^T = K Q^T (32x32x64, e4m3): lane l holds row l % 32 and keys 8 (i / 4) + 4 (l / 32) + i % 4.  O^T += V^T P^T
// (32x32x16, f16): the lane's own weights in the order it has them, V^T by the transpose read from LDS rows in that order.
__global__ __launch_bounds__(64) void chunk_kernel(ChunkDev d) {
  __shared__ __align__(16) uint8_t vs[kCST * kCD];
  const int lane = threadIdx.x, col = lane & 31, g = lane >> 5, h = blockIdx.x & 1;
  int tile = blockIdx.x >> 1, b = 0;
  Req R{0, 0, 0};
  for (;; ++b) {
    if (b >= d.B) return;
    R = req_of(d, b);
    const int n = (R.n + 3) / 4;
    if (tile < n) break;
    tile -= n;
  }
  const int pre = R.nk - R.n, i0 = 4 * tile, row_t = i0 + (col >> 3), head = h * kCG + (col & 7);
  const bool row_ok = row_t < R.n;
  const int lim = row_ok ? pre + row_t : -1;  // the row's last key
  const int nkeys = min(R.nk, pre + min(i0 + 4, R.n));
  v8i qf[4];
#pragma unroll
  for (int kb = 0; kb < 4; ++kb) {
    int w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (row_ok) {
      const size_t at = ((size_t)(R.t0 + row_t) * kCHQ + head) * kCD + 64 * kb + 32 * g;
      if (d.q8) {
        const v4i* src = reinterpret_cast<const v4i*>(static_cast<const uint8_t*>(d.q) + at);
        const v4i a = src[0], e = src[1];
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = e.x, w[5] = e.y, w[6] = e.z, w[7] = e.w;
      } else {
        const v4i* src = reinterpret_cast<const v4i*>(static_cast<const uint16_t*>(d.q) + at);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const v4i r = src[c];
#pragma unroll
          for (int j = 0; j < 2; ++j)
            w[2 * c + j] = (int)(f2e4m3x2_nan(bf_lo((uint32_t)r[2 * j]), bf_hi((uint32_t)r[2 * j])) |
                                 (f2e4m3x2_nan(bf_lo((uint32_t)r[2 * j + 1]), bf_hi((uint32_t)r[2 * j + 1])) << 16));
        }
      }
    }
    qf[kb] = v8i{w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]};
  }
  v16f o[8];
#pragma unroll
  for (int dt = 0; dt < 8; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  float m = -1e30f, l = 0.f;
  for (int k0 = 0; k0 < nkeys; k0 += kCST) {
    // V rows: LDS row r holds key 16 (r / 16) + 8 ((r % 8) / 4) + 4 ((r / 8) % 2) + r % 4, its 16-byte piece p at p ^ (r % 8);
    // a key behind the range is zero
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + (lane >> 4), p = lane & 15, key = k0 + 16 * (r >> 4) + 8 * ((r & 7) >> 2) + 4 * ((r >> 3) & 1) + (r & 3);
      v4i v = {0, 0, 0, 0};
      if (key < nkeys) v = *reinterpret_cast<const v4i*>(d.vc + ((size_t)slot_of(d, b, key) * kCHKV + h) * kCD + 16 * p);
      *reinterpret_cast<v4i*>(vs + r * kCD + 16 * (p ^ (r & 7))) = v;
    }
    __syncthreads();
    v16f s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
    const uint8_t* kr = d.kc + ((size_t)slot_of(d, b, min(k0 + col, nkeys - 1)) * kCHKV + h) * kCD + 32 * g;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      const v4i a = *reinterpret_cast<const v4i*>(kr + 64 * kb), e = *reinterpret_cast<const v4i*>(kr + 64 * kb + 16);
      s = mfma_qk(v8i{a.x, a.y, a.z, a.w, e.x, e.y, e.z, e.w}, qf[kb], s);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = k0 + 8 * (i >> 2) + 4 * g + (i & 3);
      s[i] = key > lim ? -INFINITY : s[i] * d.scale_log2;
      mx = fmaxf(mx, s[i]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float mn = fmaxf(m, mx), al = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= al;
    v8h pb[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float p = __builtin_amdgcn_exp2f(s[i] - m);
      l += p;
      pb[i >> 3][i & 7] = (_Float16)p;
    }
    const bool border = k0 + kCST - 1 > pre + i0;
    v8h vis[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) vis[i >> 3][i & 7] = k0 + 8 * (i >> 2) + 4 * g + (i & 3) <= lim ? (_Float16)1.f : (_Float16)0.f;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][i] *= al;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = 16 * c + 8 * g + ((lane & 15) >> 1), p = 2 * dt + ((lane >> 4) & 1);
        v2i w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (__attribute__((address_space(3))) v2i*)(vs + r * kCD + 16 * (p ^ (r & 7)) + 8 * (lane & 1)));
        const uint32_t n0 = nan_bytes(w.x) >> 7, n1 = nan_bytes(w.y) >> 7;
        if (border && __builtin_amdgcn_ballot_w64((n0 | n1) != 0)) {
          v16f seen;
#pragma unroll
          for (int i = 0; i < 16; ++i) seen[i] = 0.f;
          seen = __builtin_amdgcn_mfma_f32_32x32x16_f16(widen8(n0 * 0x38, n1 * 0x38), vis[c], seen, 0, 0, 0);
          w = v2i{(int)(w.x & ~(n0 * 0xff)), (int)(w.y & ~(n1 * 0xff))};
#pragma unroll
          for (int i = 0; i < 16; ++i) o[dt][i] = seen[i] > 0.f ? __builtin_nanf("") : o[dt][i];
        }
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(widen8(w.x, w.y), pb[c], o[dt], 0, 0, 0);
      }
    }
  }
  l += __shfl_xor(l, 32);
  const float il = l > 0.f ? 1.f / l : l;  // (NaN stays)
  if (!row_ok) return;
  uint16_t* dst = d.out + ((size_t)(R.t0 + row_t) * kCHQ + head) * kCD + 4 * g;
#pragma unroll
  for (int dt = 0; dt < 8; ++dt)
#pragma unroll
    for (int a = 0; a < 4; ++a)
      *reinterpret_cast<uint2*>(dst + 32 * dt + 8 * a) = make_uint2(pack_bf2(o[dt][4 * a] * il, o[dt][4 * a + 1] * il),
                                                                    pack_bf2(o[dt][4 * a + 2] * il, o[dt][4 * a + 3] * il));
}

}  // namespace
}  // namespace q36

using namespace q36;

extern "C" size_t q36_attn_chunk_workspace_bytes(void) { return 256; }

extern "C" int q36_attn_chunk(const q36_chunk_args* a, q36_stream_t stream) {
  Q36_REQUIRE(a != nullptr, "q36_attn_chunk: null args");
  Q36_REQUIRE(a->HQ == kCHQ && a->HKV == kCHKV && a->D == kCD, "q36_attn_chunk: HQ=%d HKV=%d D=%d unsupported (this build: 16 / 2 / 256)",
              a->HQ, a->HKV, a->D);
  Q36_REQUIRE(a->B >= 1 && a->B <= 65535 && a->T >= 1 && a->T <= (1 << 20), "q36_attn_chunk: B=%d T=%d out of range", a->B, a->T);
  Q36_REQUIRE(a->page_size >= 1 && a->page_size <= 1024 && (a->page_size & (a->page_size - 1)) == 0,
              "q36_attn_chunk: page_size=%d must be a power of two up to 1024", a->page_size);
  Q36_REQUIRE(a->pt_stride >= 1 && a->pt_stride <= (1 << 27) / a->page_size, "q36_attn_chunk: pt_stride=%d of pages of %d out of range",
              a->pt_stride, a->page_size);
  Q36_REQUIRE(a->num_slots >= 1 && a->num_slots < ((int64_t)1 << 31), "q36_attn_chunk: num_slots=%lld out of range",
              (long long)a->num_slots);
  Q36_REQUIRE(a->q && a->k_cache && a->v_cache && a->page_table && a->seqlens && a->qsl && a->out && a->workspace,
              "q36_attn_chunk: a required pointer is null");
  Q36_REQUIRE(aligned16(a->q) && aligned16(a->k_cache) && aligned16(a->v_cache) && aligned16(a->out) &&
                  (reinterpret_cast<uintptr_t>(a->workspace) & 255u) == 0,
              "q36_attn_chunk: q, out and the caches must be 16-byte and workspace 256-byte aligned");
  Q36_REQUIRE(a->workspace_bytes >= q36_attn_chunk_workspace_bytes(), "q36_attn_chunk: workspace of %zu bytes < %zu required",
              a->workspace_bytes, q36_attn_chunk_workspace_bytes());
  int sh = 0;
  while ((1 << sh) < a->page_size) ++sh;
  const ChunkDev d{a->B, a->T, sh, a->pt_stride, a->q_e4m3, a->num_slots, a->q, static_cast<const uint8_t*>(a->k_cache),
                   static_cast<const uint8_t*>(a->v_cache), a->page_table, a->seqlens, a->qsl, static_cast<uint16_t*>(a->out),
                   a->scale * 1.44269504088896340736f};
  chunk_kernel<<<2 * (unsigned)(a->T / 4 + a->B), 64, 0, static_cast<hipStream_t>(stream)>>>(d);
  return check_launch("q36_attn_chunk");
}
