// The attention layer's front behind the q/gate/k/v projection: per-head Gemma RMSNorm on q and k, neox RoPE on the
// first 64 of 256 dims with positions of one or several axes (time, height, width), the query rows (bf16, or e4m3 as the
// chunk attention reads them), the gate rows and the new e4m3 K / V rows in the cache.
//
// Reference behaviour (R = qwen36_nodes_kb34, L = R/qwen36_layer): L/qk_attn_verify.cu:765-797 attn_prefill_front
// (norm, RoPE, q8 out, K and V cache rows; one position a token).
//
//   y = x * rsqrt(mean x^2 + eps) * (1 + w);  (y_i, y_{i+32}) turned by the angle of pair i at position[axis(i)]
//
// Everything is formed in fp32 and rounded once.  Bytes bound it: 18 KB read and 13 or 17 KB written a token.  8192 tokens
// with bf16 queries (294 MB) take 50 us on the GPU, 5.8 TB/s (a copy of 2 GiB, both directions counted, 4.75), 1777 with
// e4m3 ones and three axes (56 MB) 17 us, one token 4 us, the launch.
#include "q36_device.h"
#include "q36_host.h"

namespace q36 {
namespace {

constexpr int kFItems = 18;  // pieces of a token's row: 16 heads of q and gate, 2 of k and v
struct FrontDev {
  int T, max_pos, axes;
  int64_t ld, pos_stride;
  uint64_t axis_map;
  const uint16_t* qkv;
  const uint16_t* q_norm_w;
  const uint16_t* k_norm_w;
  const float* cos_sin;
  const int32_t* positions;
  void* q;
  uint16_t* gate;
  const int64_t* out_loc;
  uint8_t* kc;
  uint8_t* vc;
  int64_t num_slots;
  float eps;
};

// A wave takes three of a token's pieces.  Lanes 0-31 hold a head of q (or k), 8 consecutive dims a lane, lanes 32-63 its
// companion (the gate, or v): one contiguous 1 KB load for a head of q and its gate.  MULTI: the pairs' positions differ by axis,
// so a lane's cosines and sines come one by one, once a wave.  Pieces a wave, us a call (one / three / nine): 8192 tokens of one
// axis 67.9 / 53.5 / 57.6, 1777 of three axes 20.4 / 17.4 / 18.7, 4000 of three axes 40.7 / 31.3 / 31.8; from 1 token to 1000
// the call's own launch hides them all.
constexpr int IPW = 3, WPT = kFItems / IPW;  // pieces of a wave, WPT apart; waves a token
template <bool MULTI, bool Q8>
__global__ __launch_bounds__(256) void front_kernel(FrontDev d) {
  const int64_t wv = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (wv >= (int64_t)d.T * WPT) return;
  const int t = __builtin_amdgcn_readfirstlane((int)(wv / WPT)), h0 = __builtin_amdgcn_readfirstlane((int)(wv % WPT));
  const int half = lane >> 5, j = lane & 31;
  const uint16_t* const row = d.qkv + (size_t)t * d.ld;
  // the token's positions, by scalar loads ahead of its row's (4000 tokens of three axes 33 -> 31 us a call)
  typedef __attribute__((address_space(4))) const int32_t* Scalars;
  const Scalars ps = (Scalars)(uintptr_t)(d.positions + t);
  int at[4];
#pragma unroll
  for (int a = 0; a < (MULTI ? 4 : 1); ++a) at[a] = min(max(ps[a < d.axes ? a * d.pos_stride : 0], 0), d.max_pos - 1);
  v4i raw[IPW];
#pragma unroll
  for (int k = 0; k < IPW; ++k) {
    const int h = h0 + WPT * k;
    const int col = h < 16 ? h * 512 + half * 256 + 8 * j : (half ? 8704 : 8192) + (h - 16) * 256 + 8 * j;
    raw[k] = *reinterpret_cast<const v4i*>(row + col);
  }
  const v4i qw = *reinterpret_cast<const v4i*>(d.q_norm_w + 8 * j), kw = *reinterpret_cast<const v4i*>(d.k_norm_w + 8 * j);
  const int64_t slot = d.out_loc ? d.out_loc[t] : -1;
  // lanes j < 8 turn dims 8 j .. 8 j + 7 by the pairs 8 (j & 3) + e
  const bool normed = half == 0, rot = normed && j < 8;
  float c[8] = {}, s[8] = {};
  if constexpr (MULTI) {
    if (rot) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = 8 * (j & 3) + e, axis = (int)(d.axis_map >> (2 * i)) & 3;
        const int pos = axis & 2 ? (axis & 1 ? at[3] : at[2]) : axis & 1 ? at[1] : at[0];
        c[e] = d.cos_sin[(size_t)pos * 64 + i];
        s[e] = d.cos_sin[(size_t)pos * 64 + 32 + i];
      }
    }
  } else {
    const int pos = at[0];
    const float* cs = d.cos_sin + (size_t)pos * 64 + 8 * (j & 3);
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const v4f a = *reinterpret_cast<const v4f*>(cs + e), b = *reinterpret_cast<const v4f*>(cs + 32 + e);
#pragma unroll
      for (int i = 0; i < 4; ++i) c[e + i] = a[i], s[e + i] = b[i];
    }
  }
  const float sg = j < 4 ? -1.f : 1.f;
#pragma unroll
  for (int k = 0; k < IPW; ++k) {
    const int h = h0 + WPT * k;
    const bool qhead = h < 16;
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf_lo((uint32_t)raw[k][i]);
      x[2 * i + 1] = bf_hi((uint32_t)raw[k][i]);
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
    ss += xor_swz<16>(ss);
    ss += xor_swz<8>(ss);
    ss += xor_swz<4>(ss);
    ss += xor_swz<2>(ss);
    ss += xor_swz<1>(ss);
    const float inv = 1.f / sqrtf(ss / 256.f + d.eps);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = (uint32_t)(qhead ? qw[i] : kw[i]);
      const float a = (x[2 * i] * inv) * (bf_lo(w) + 1.f), b = (x[2 * i + 1] * inv) * (bf_hi(w) + 1.f);
      x[2 * i] = normed ? a : x[2 * i];
      x[2 * i + 1] = normed ? b : x[2 * i + 1];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float other = xor_swz<4>(x[e]);
      const float r = __builtin_fmaf(x[e], c[e], (sg * other) * s[e]);
      x[e] = rot ? r : x[e];
    }
    const auto codes = [&] {
      return make_uint2(f2e4m3x2_nan(x[0], x[1]) | (f2e4m3x2_nan(x[2], x[3]) << 16),
                        f2e4m3x2_nan(x[4], x[5]) | (f2e4m3x2_nan(x[6], x[7]) << 16));
    };
    if (qhead) {
      const size_t at = ((size_t)t * 16 + h) * 256 + 8 * j;
      if (!normed) {
        if (d.gate) *reinterpret_cast<v4i*>(d.gate + at) = raw[k];
      } else if constexpr (Q8) {
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(d.q) + at) = codes();
      } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(d.q) + at) = make_uint4(
            pack_bf2_hw(x[0], x[1]), pack_bf2_hw(x[2], x[3]), pack_bf2_hw(x[4], x[5]), pack_bf2_hw(x[6], x[7]));
      }
    } else if (slot >= 0 && slot < d.num_slots) {
      *reinterpret_cast<uint2*>((normed ? d.kc : d.vc) + ((size_t)slot * 2 + (h - 16)) * 256 + 8 * j) = codes();
    }
  }
}

}  // namespace
}  // namespace q36

using namespace q36;

extern "C" int q36_attn_front(const q36_attn_front_args* a, q36_stream_t stream) {
  Q36_REQUIRE(a != nullptr, "q36_attn_front: null args");
  Q36_REQUIRE(a->T >= 1 && a->T <= (1 << 20), "q36_attn_front: T=%d out of range", a->T);
  Q36_REQUIRE(a->max_pos >= 1, "q36_attn_front: max_pos=%d", a->max_pos);
  Q36_REQUIRE(a->axes >= 1 && a->axes <= 4, "q36_attn_front: axes=%d (1 .. 4)", a->axes);
  for (int i = 0; i < 32; ++i)
    Q36_REQUIRE((int)((uint64_t)a->axis_map >> (2 * i) & 3) < a->axes, "q36_attn_front: pair %d on axis %d of %d", i,
                (int)((uint64_t)a->axis_map >> (2 * i) & 3), a->axes);
  Q36_REQUIRE(a->axes == 1 || a->pos_stride >= a->T, "q36_attn_front: positions of stride %lld for T=%d",
              (long long)a->pos_stride, a->T);
  Q36_REQUIRE(a->qkv_ld >= 9216 && a->qkv_ld % 8 == 0, "q36_attn_front: qkv_ld=%lld must be a multiple of 8 from 9216 on",
              (long long)a->qkv_ld);
  Q36_REQUIRE(a->qkv && a->q_norm_w && a->k_norm_w && a->cos_sin && a->positions && a->q,
              "q36_attn_front: a required pointer is null");
  Q36_REQUIRE((a->out_loc == nullptr) == (a->k_cache == nullptr) && (a->k_cache == nullptr) == (a->v_cache == nullptr),
              "q36_attn_front: out_loc, k_cache and v_cache go together");
  Q36_REQUIRE(!a->out_loc || (a->num_slots >= 1 && a->num_slots < ((int64_t)1 << 31)),
              "q36_attn_front: num_slots=%lld out of range", (long long)a->num_slots);
  Q36_REQUIRE(aligned16(a->qkv) && aligned16(a->q_norm_w) && aligned16(a->k_norm_w) && aligned16(a->cos_sin) &&
                  aligned16(a->gate) && (reinterpret_cast<uintptr_t>(a->q) & (a->q_e4m3 ? 7u : 15u)) == 0 &&
                  (reinterpret_cast<uintptr_t>(a->k_cache) & 7u) == 0 && (reinterpret_cast<uintptr_t>(a->v_cache) & 7u) == 0,
              "q36_attn_front: qkv, the norm weights, cos_sin, gate and bf16 q must be 16-byte, e4m3 q and the caches "
              "8-byte aligned");
  const FrontDev d{a->T, a->max_pos, a->axes, a->qkv_ld, a->pos_stride, (uint64_t)a->axis_map,
                   static_cast<const uint16_t*>(a->qkv), static_cast<const uint16_t*>(a->q_norm_w),
                   static_cast<const uint16_t*>(a->k_norm_w), a->cos_sin, a->positions, a->q,
                   static_cast<uint16_t*>(a->gate), a->out_loc, static_cast<uint8_t*>(a->k_cache),
                   static_cast<uint8_t*>(a->v_cache), a->num_slots, a->eps};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool multi = a->axis_map != 0, q8 = a->q_e4m3 != 0;
  const unsigned grid = (unsigned)(((int64_t)a->T * WPT + 3) / 4);
  if (multi)
    q8 ? front_kernel<true, true><<<grid, 256, 0, st>>>(d) : front_kernel<true, false><<<grid, 256, 0, st>>>(d);
  else
    q8 ? front_kernel<false, true><<<grid, 256, 0, st>>>(d) : front_kernel<false, false><<<grid, 256, 0, st>>>(d);
  return check_launch("q36_attn_front");
}
