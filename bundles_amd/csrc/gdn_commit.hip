// Commit of a verified draft window to the recurrent state over the ReplaySSM ring: the conv state goes to the accepted
// position, and where the ring has no room for the next window its entries are folded into the checkpoint.  (The reference
// leaves both to its serving engine; the pools are those of its verify kernel, R/qwen36_layer/qk_gdn_verify.cu:841-919.)
//
//   n = write_pos + accepted; conv_state = window[:, accepted - 1 .. accepted + 1]
//   n + room > 16:  h0 <- e^{G_n} h0 + sum_{c < n} e^{G_n - G_c} (d + dlo)_c (k + klo)_c^T,  G_c = g_0 + .. + g_c
//
// Bytes bound it: a folded request moves 4 MB of checkpoint and up to 0.4 MB of ring, the others 0.15 MB.  256 requests of 8
// drafts (597 MB): 133 us, 4.5 TB/s (a copy moves 4.75).
#include "q36_device.h"
#include "q36_host.h"

namespace q36 {
namespace {

constexpr int CK = 128, CV = 128, CHK = 16, CHV = 32, CQKV = 8192, CL = 16;
constexpr int kConvParts = 16, kConvCh = CQKV / kConvParts;  // workgroups a request for the conv state, channels of each

struct CommitDev {
  int B, T, room, slots, rslots, wslots, idx_i64;
  uint16_t* conv_state;
  int64_t cs_slot;
  const uint16_t* window;
  int64_t win_slot;
  float* h0;
  const uint16_t* d;
  const uint16_t* dlo;
  int64_t d_slot, dlo_slot;
  const uint16_t* k;
  const uint16_t* klo;
  int64_t k_slot, klo_slot;
  const float* g;
  int64_t g_slot;
  const void* state_idx;
  const void* replay_idx;
  const void* win_idx;
  const void* accepted;
  int32_t* write_pos;
  int32_t* cache_base;
};

__device__ __forceinline__ int64_t index_at(const void* p, int i64, int r) {
  return i64 ? static_cast<const int64_t*>(p)[r] : (int64_t)static_cast<const int32_t*>(p)[r];
}

// A request's slots and cursors; false: a padded request (an index outside its pool, nothing accepted).
struct Request {
  int64_t slot, rp, ws;
  int acc, n, base;
  bool fold;
};
__device__ __forceinline__ bool request(const CommitDev& d, int r, Request& q) {
  q.slot = index_at(d.state_idx, d.idx_i64 & 1, r);
  q.rp = index_at(d.replay_idx, d.idx_i64 & 2, r);
  q.ws = index_at(d.win_idx, d.idx_i64 & 4, r);
  const int64_t acc = index_at(d.accepted, d.idx_i64 & 8, r);
  if (q.slot < 0 || q.slot >= d.slots || q.rp < 0 || q.rp >= d.rslots || q.ws < 0 || q.ws >= d.wslots || acc < 1) return false;
  q.acc = (int)(acc < d.T ? acc : d.T);
  const int wp = min(max(d.write_pos[q.rp], 0), CL);
  q.base = d.cache_base[q.rp] & (CL - 1);
  q.n = min(wp + q.acc, CL);  // (entries past the ring's end were never appended)
  q.fold = q.n + d.room > CL;
  return true;
}

__global__ __launch_bounds__(256) void commit_kernel(CommitDev d) {
  __shared__ __attribute__((aligned(16))) float dl[CV][CL];  // a head's d entries by value row, decayed
  __shared__ __attribute__((aligned(16))) uint16_t win[kConvCh * 10];
  const int r = blockIdx.x / (CHV + kConvParts), part = blockIdx.x % (CHV + kConvParts), tid = threadIdx.x;
  Request q;
  if (!request(d, r, q)) return;
  if (part >= CHV) {  // ---- 512 channels of the conv state
    const int ch0 = (part - CHV) * kConvCh, W = d.T + 2;
    const uint16_t* src = d.window + q.ws * d.win_slot + (int64_t)ch0 * W;
    for (int i = tid; i < kConvCh * W / 8; i += 256)
      *reinterpret_cast<v4i*>(win + 8 * i) = *reinterpret_cast<const v4i*>(src + 8 * i);
    __syncthreads();
    if (tid < kConvCh * 3 / 8) {
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const int e0 = 8 * tid + i, e1 = e0 + 1;
        o[i >> 1] = (uint32_t)win[e0 / 3 * W + q.acc - 1 + e0 % 3] | ((uint32_t)win[e1 / 3 * W + q.acc - 1 + e1 % 3] << 16);
      }
      *reinterpret_cast<v4i*>(d.conv_state + q.slot * d.cs_slot + (int64_t)ch0 * 3 + 8 * tid) = __builtin_bit_cast(v4i, o);
    }
    return;
  }
  if (!q.fold) return;
  // ---- a value head's checkpoint.  Entry c lies at physical slot (base + c) & 15; its decay is the sum of the gates
  // behind it, last first
  const int hv = part, hk = hv / 2;
  const float* g = d.g + q.rp * d.g_slot + hv * CL;
  float fade[CL], run = 0.f;
#pragma unroll
  for (int c = CL - 1; c >= 0; --c) {
    const float gc = g[(q.base + c) & (CL - 1)];
    fade[c] = c < q.n ? expf_q(run) : 0.f;
    run = c < q.n ? run + gc : run;
  }
  const float all = expf_q(run);
  const uint16_t* dh = d.d + q.rp * d.d_slot + (int64_t)hv * CL * CV;
  const uint16_t* dw = d.dlo + q.rp * d.dlo_slot + (int64_t)hv * CL * CV;
  if (tid < CV) {
#pragma unroll
    for (int c = 0; c < CL; ++c) {
      const int at = ((q.base + c) & (CL - 1)) * CV + tid;
      const float v = bf2f(dh[at]) + bf2f(dw[at]);
      dl[tid][c] = c < q.n ? v * fade[c] : 0.f;
    }
  }
  // four key columns of every entry in registers
  const int col = (tid & 31) * 4, r0 = tid >> 5;
  const uint16_t* kh = d.k + q.rp * d.k_slot + (int64_t)hk * CL * CK + col;
  const uint16_t* kw = d.klo + q.rp * d.klo_slot + (int64_t)hk * CL * CK + col;
  v4f kk[CL];
#pragma unroll
  for (int c = 0; c < CL; ++c) {
    const int at = ((q.base + c) & (CL - 1)) * CK;
    const v2i hi = *reinterpret_cast<const v2i*>(kh + at), lo = *reinterpret_cast<const v2i*>(kw + at);
    v4f v;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[2 * i] = bf_lo((uint32_t)hi[i]) + bf_lo((uint32_t)lo[i]);
      v[2 * i + 1] = bf_hi((uint32_t)hi[i]) + bf_hi((uint32_t)lo[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) kk[c][i] = c < q.n ? v[i] : 0.f;
  }
  __syncthreads();
  float* h = d.h0 + (q.slot * CHV + hv) * (int64_t)(CV * CK) + col;
#pragma unroll 4
  for (int i = 0; i < CV / 8; ++i) {
    const int row = r0 + 8 * i;
    v4f s = *reinterpret_cast<const v4f*>(h + row * CK);
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] *= all;
#pragma unroll
    for (int c4 = 0; c4 < CL; c4 += 4) {
      const v4f dv = *reinterpret_cast<const v4f*>(&dl[row][c4]);
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = __builtin_fmaf(dv[c], kk[c4 + c][j], s[j]);
    }
    *reinterpret_cast<v4f*>(h + row * CK) = s;
  }
}

// The ring's cursors, behind every workgroup that reads them.
__global__ __launch_bounds__(256) void commit_advance_kernel(CommitDev d) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  Request q;
  if (r >= d.B || !request(d, r, q)) return;
  d.write_pos[q.rp] = q.fold ? 0 : q.n;
  if (q.fold) d.cache_base[q.rp] = (q.base + q.n) & (CL - 1);
}

}  // namespace
}  // namespace q36

using namespace q36;

extern "C" int q36_gdn_ring_commit(const q36_gdn_commit_args* a, q36_stream_t stream) {
  Q36_REQUIRE(a != nullptr, "q36_gdn_ring_commit: null args");
  Q36_REQUIRE(a->B >= 0 && a->B <= 65535, "q36_gdn_ring_commit: B=%d out of range", a->B);
  Q36_REQUIRE(a->T >= 1 && a->T <= 8, "q36_gdn_ring_commit: T=%d must be in [1,8]", a->T);
  Q36_REQUIRE(a->room >= 0 && a->room <= CL, "q36_gdn_ring_commit: room=%d must be in [0,16]", a->room);
  if (a->B == 0) return Q36_OK;
  Q36_REQUIRE(a->conv_state && a->window && a->h0 && a->d_ring && a->dlo_ring && a->k_ring && a->klo_ring && a->g_ring &&
                  a->state_idx && a->replay_idx && a->win_idx && a->accepted && a->write_pos && a->cache_base,
              "q36_gdn_ring_commit: a required pointer is null");
  Q36_REQUIRE(a->slots >= 1 && a->rslots >= 1 && a->wslots >= 1, "q36_gdn_ring_commit: slots=%d rslots=%d wslots=%d",
              a->slots, a->rslots, a->wslots);
  Q36_REQUIRE(a->cs_slot >= CQKV * 3 && a->cs_slot % 8 == 0, "q36_gdn_ring_commit: conv_state slot stride %lld",
              (long long)a->cs_slot);
  Q36_REQUIRE(a->win_slot >= (int64_t)CQKV * (a->T + 2) && a->win_slot % 8 == 0,
              "q36_gdn_ring_commit: window slot stride %lld must be >= 8192 x %d and a multiple of 8", (long long)a->win_slot,
              a->T + 2);
  Q36_REQUIRE(a->d_slot >= CHV * CL * CV && a->dlo_slot >= CHV * CL * CV && a->d_slot % 8 == 0 && a->dlo_slot % 8 == 0,
              "q36_gdn_ring_commit: d ring slot strides must be >= 32 x 16 x 128 and multiples of 8");
  Q36_REQUIRE(a->k_slot >= CHK * CL * CK && a->klo_slot >= CHK * CL * CK && a->k_slot % 8 == 0 && a->klo_slot % 8 == 0,
              "q36_gdn_ring_commit: k ring slot strides must be >= 16 x 16 x 128 and multiples of 8");
  Q36_REQUIRE(a->g_slot >= CHV * CL && a->g_slot % 4 == 0, "q36_gdn_ring_commit: g ring slot stride %lld", (long long)a->g_slot);
  Q36_REQUIRE(aligned16(a->h0) && aligned16(a->conv_state) && aligned16(a->window) && aligned16(a->d_ring) &&
                  aligned16(a->dlo_ring) && aligned16(a->k_ring) && aligned16(a->klo_ring) && aligned16(a->g_ring),
              "q36_gdn_ring_commit: h0, conv_state, window and the rings must be 16-byte aligned");
  CommitDev d{a->B, a->T, a->room, a->slots, a->rslots, a->wslots, a->idx_i64,
              static_cast<uint16_t*>(a->conv_state), a->cs_slot, static_cast<const uint16_t*>(a->window), a->win_slot, a->h0,
              static_cast<const uint16_t*>(a->d_ring), static_cast<const uint16_t*>(a->dlo_ring), a->d_slot, a->dlo_slot,
              static_cast<const uint16_t*>(a->k_ring), static_cast<const uint16_t*>(a->klo_ring), a->k_slot, a->klo_slot,
              a->g_ring, a->g_slot, a->state_idx, a->replay_idx, a->win_idx, a->accepted, a->write_pos, a->cache_base};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  commit_kernel<<<(unsigned)a->B * (CHV + kConvParts), 256, 0, st>>>(d);
  if (a->advance) commit_advance_kernel<<<(a->B + 255) / 256, 256, 0, st>>>(d);
  return check_launch("q36_gdn_ring_commit");
}
