// The recurrent layer's prompt: causal conv + SiLU, q/k L2 norm, gates, the gated delta rule over any number of new tokens
// a request, the gated RMSNorm of the output; conv state and recurrent state carried in the engine's pools.  (The
// reference leaves prompts to its engine's kernels; the layer is that of its verify kernel, R/qwen36_layer/
// qk_gdn_verify.cu:238-247 conv, :575-581 norms, :616-622 gates, :684-762 recurrence, :786-791 output norm.)
//
//   S <- e^g S;  u = beta (v - S k);  S <- S + u k^T;  o = S q;  out = o rsqrt(mean o^2 + eps) w silu(z)
//
// Everything is formed in fp32 and rounded once.  (The verify kernels round the conv's tap products, its output and o to
// bf16, as the reference's does.)
#include "q36_device.h"
#include "q36_host.h"

namespace q36 {
namespace {

constexpr int PK = 128, PV = 128, PHK = 16, PHV = 32, PQKV = 8192, PZ = PHV * PV;
constexpr int kGroup = 8;  // tokens whose conv, norms and gates are formed at once

struct PromptDev {
  int B, rows, slots, idx_i64, dt_f32;
  float eps, scale;
  const uint16_t* mixed;
  const uint16_t* z;
  const uint16_t* a;
  const uint16_t* b;
  uint16_t* conv_state;
  int64_t cs_slot;
  const uint16_t* conv_w;
  const float* A_log;
  const void* dt_bias;
  float* h0;
  const int32_t* qsl;
  const void* state_idx;
  const int32_t* prefix;
  const uint16_t* norm_w;
  uint16_t* out;
  uint8_t* oq;
  float* oqs;
};

// Request r's rows, inside the batch whatever qsl holds, and its slot (-1: none).
__device__ __forceinline__ void request_of(const PromptDev& d, int r, int& t0, int& n, int64_t& slot, bool& old) {
  const int lo = min(max(d.qsl[r], 0), d.rows), hi = min(max(d.qsl[r + 1], 0), d.rows);
  t0 = lo, n = max(hi - lo, 0);
  const int64_t s = d.idx_i64 ? static_cast<const int64_t*>(d.state_idx)[r] : (int64_t)static_cast<const int32_t*>(d.state_idx)[r];
  slot = s >= 0 && s < d.slots ? s : -1;
  old = d.prefix == nullptr || d.prefix[r] > 0;
}

__device__ __forceinline__ float silu(float x) { return x / (1.f + expf_q(-x)); }
// log(1 + e^x)
__device__ __forceinline__ float softplus(float x) { return x > 20.f ? x : log1pf(expf_q(x)); }

// One 512-thread workgroup a (request, key head): both value heads' states in registers, rows (tid / 8) + 64 j (head j / 2),
// columns 32 jj + 4 (tid % 8) .. + 3; a row's dot is 16 local fma and three steps over its 8 threads.
__global__ __launch_bounds__(512) void prompt_steps_kernel(PromptDev d) {
  __shared__ __attribute__((aligned(16))) float qs[kGroup][PK], ks[kGroup][PK];
  __shared__ float vs[kGroup][2 * PV], os[kGroup][2 * PV];
  __shared__ float eg[kGroup][2], beta[kGroup][2];
  const int r = blockIdx.x / PHK, hk = blockIdx.x % PHK;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int t0, n;
  int64_t slot;
  bool old;
  request_of(d, r, t0, n, slot, old);
  if (n == 0) return;
  if (slot < 0) {  // a padded request: zero rows
    for (int i = tid; i < n * 64; i += 512) {
      const int64_t o = (int64_t)(t0 + (i >> 6)) * PZ + hk * 2 * PV + (i & 63) * 4;
      *reinterpret_cast<v2i*>(d.out + o) = v2i{0, 0};
      if (d.oq) {
        *reinterpret_cast<uint32_t*>(d.oq + o) = 0u;
        if ((i & 63) < 2) d.oqs[(int64_t)(t0 + (i >> 6)) * PHV + 2 * hk + (i & 63)] = 0.f;
      }
    }
    return;
  }
  const int r0 = tid >> 3, c8 = tid & 7;
  float* const hp = d.h0 + (slot * PHV + 2 * hk) * (int64_t)(PV * PK);
  v4f st[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int jj = 0; jj < 4; ++jj)
      st[j][jj] = old ? *reinterpret_cast<const v4f*>(hp + (r0 + 64 * j) * PK + 32 * jj + 4 * c8) : v4f{0.f, 0.f, 0.f, 0.f};
  // one conv channel a thread: q and k of the key head, v of its value heads
  const int ch = tid < 256 ? (tid >> 7) * (PHK * PK) + hk * PK + (tid & 127) : 2 * PHK * PK + hk * 2 * PV + (tid - 256);
  uint16_t* const cs = d.conv_state + slot * d.cs_slot + (int64_t)ch * 3;
  float w0 = old ? bf2f(cs[0]) : 0.f, w1 = old ? bf2f(cs[1]) : 0.f, w2 = old ? bf2f(cs[2]) : 0.f;
  float cw[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) cw[i] = bf2f(d.conv_w[(int64_t)ch * 4 + i]);
  for (int g0 = 0; g0 < n; g0 += kGroup) {
    const int G = min(kGroup, n - g0);
    for (int t = 0; t < G; ++t) {
      const float x = bf2f(d.mixed[(int64_t)(t0 + g0 + t) * PQKV + ch]);
      float y = w0 * cw[0];
      y = __builtin_fmaf(w1, cw[1], y);
      y = __builtin_fmaf(w2, cw[2], y);
      y = __builtin_fmaf(x, cw[3], y);
      w0 = w1, w1 = w2, w2 = x;
      y = silu(y);
      if (tid < 128) qs[t][tid] = y;
      else if (tid < 256) ks[t][tid - 128] = y;
      else vs[t][tid - 256] = y;
    }
    if (tid < 2 * G) {
      const int t = tid >> 1, h = 2 * hk + (tid & 1);
      const int64_t o = (int64_t)(t0 + g0 + t) * PHV + h;
      const float dt = d.dt_f32 ? static_cast<const float*>(d.dt_bias)[h] : bf2f(static_cast<const uint16_t*>(d.dt_bias)[h]);
      eg[t][tid & 1] = expf_q(-expf_q(d.A_log[h]) * softplus(bf2f(d.a[o]) + dt));
      beta[t][tid & 1] = sigmoid_q(bf2f(d.b[o]));
    }
    __syncthreads();
    for (int p = wave; p < 2 * G; p += 8) {
      float* x = (p & 1) ? ks[p >> 1] : qs[p >> 1];
      const float a0 = x[lane], a1 = x[lane + 64];
      float rr = 1.f / sqrtf(wave_sum_bfly(a0 * a0 + a1 * a1) + 1e-6f);
      if (!(p & 1)) rr = rr * d.scale;
      x[lane] = a0 * rr;
      x[lane + 64] = a1 * rr;
    }
    __syncthreads();
    for (int t = 0; t < G; ++t) {
      v4f kk[4], qq[4];
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        kk[jj] = *reinterpret_cast<const v4f*>(&ks[t][32 * jj + 4 * c8]);
        qq[jj] = *reinterpret_cast<const v4f*>(&qs[t][32 * jj + 4 * c8]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = eg[t][j >> 1];
        float kv = 0.f, ov = 0.f;
#pragma unroll
        for (int jj = 0; jj < 4; ++jj)
#pragma unroll
          for (int i = 0; i < 4; ++i) kv = __builtin_fmaf(st[j][jj][i], kk[jj][i], kv);
        kv = kv + lane_xor<1>(kv);
        kv = kv + lane_xor<2>(kv);
        kv = kv + lane_xor<4>(kv);
        const float u = beta[t][j >> 1] * (vs[t][r0 + 64 * j] - e * kv);
#pragma unroll
        for (int jj = 0; jj < 4; ++jj)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            st[j][jj][i] = __builtin_fmaf(e, st[j][jj][i], u * kk[jj][i]);
            ov = __builtin_fmaf(st[j][jj][i], qq[jj][i], ov);
          }
        ov = ov + lane_xor<1>(ov);
        ov = ov + lane_xor<2>(ov);
        ov = ov + lane_xor<4>(ov);
        if (c8 == 0) os[t][r0 + 64 * j] = ov;
      }
    }
    __syncthreads();
    for (int p = wave; p < 2 * G; p += 8) {
      const int t = p >> 1, h = p & 1;
      const int64_t row = t0 + g0 + t, o = row * PZ + (2 * hk + h) * PV;
      const float o0 = os[t][h * PV + lane], o1 = os[t][h * PV + lane + 64];
      const float rstd = 1.f / sqrtf(wave_sum_bfly(o0 * o0 + o1 * o1) / (float)PV + d.eps);
      const float y0 = o0 * rstd * bf2f(d.norm_w[lane]) * silu(bf2f(d.z[o + lane]));
      const float y1 = o1 * rstd * bf2f(d.norm_w[lane + 64]) * silu(bf2f(d.z[o + lane + 64]));
      const uint32_t y = pack_bf2(y0, y1);
      d.out[o + lane] = (uint16_t)y;
      d.out[o + lane + 64] = (uint16_t)(y >> 16);
      if (d.oq) {
        const float f0 = bf_lo(y), f1 = bf_hi(y);
        const float m = wave_max(fmaxf(fabsf(f0), fabsf(f1)));
        const float inv = m > 0.f ? 448.f / m : 0.f;
        const uint32_t cd = f2e4m3x2_hw(f0 * inv, f1 * inv);
        d.oq[o + lane] = (uint8_t)(cd & 0xffu);
        d.oq[o + lane + 64] = (uint8_t)((cd >> 8) & 0xffu);
        if (lane == 0) d.oqs[row * PHV + 2 * hk + h] = m / 448.f;
      }
    }
  }
  cs[0] = (uint16_t)(__float_as_uint(w0) >> 16);
  cs[1] = (uint16_t)(__float_as_uint(w1) >> 16);
  cs[2] = (uint16_t)(__float_as_uint(w2) >> 16);
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) *reinterpret_cast<v4f*>(hp + (r0 + 64 * j) * PK + 32 * jj + 4 * c8) = st[j][jj];
}

}  // namespace
}  // namespace q36

using namespace q36;

extern "C" size_t q36_gdn_prompt_workspace_bytes(int32_t rows, int32_t B) {
  if (rows < 1 || B < 1) return 0;
  return 256;
}

extern "C" int q36_gdn_prompt(const q36_gdn_prompt_args* a, q36_stream_t stream) {
  Q36_REQUIRE(a != nullptr, "q36_gdn_prompt: null args");
  Q36_REQUIRE(a->B >= 0 && a->B <= 65535, "q36_gdn_prompt: B=%d out of range", a->B);
  Q36_REQUIRE(a->rows >= 0 && a->rows <= (1 << 20), "q36_gdn_prompt: rows=%d out of range", a->rows);
  if (a->B == 0 || a->rows == 0) return Q36_OK;
  Q36_REQUIRE(a->mixed && a->z && a->a && a->b && a->conv_state && a->conv_w && a->A_log && a->dt_bias && a->h0 && a->qsl &&
                  a->state_idx && a->norm_w && a->out && a->workspace,
              "q36_gdn_prompt: a required pointer is null");
  Q36_REQUIRE(a->slots >= 1, "q36_gdn_prompt: slots=%d", a->slots);
  Q36_REQUIRE(a->cs_slot >= PQKV * 3 && a->cs_slot % 8 == 0, "q36_gdn_prompt: conv_state slot stride %lld", (long long)a->cs_slot);
  Q36_REQUIRE(aligned16(a->mixed) && aligned16(a->z) && aligned16(a->conv_state) && aligned16(a->conv_w) && aligned16(a->h0) &&
                  aligned16(a->out),
              "q36_gdn_prompt: mixed, z, conv_state, conv_w, h0 and out must be 16-byte aligned");
  Q36_REQUIRE((reinterpret_cast<uintptr_t>(a->dt_bias) & 3u) == 0, "q36_gdn_prompt: dt_bias must be 4-byte aligned");
  Q36_REQUIRE((a->oq == nullptr) == (a->oqs == nullptr), "q36_gdn_prompt: oq and oqs go together");
  Q36_REQUIRE(!a->oq || (aligned16(a->oq) && (reinterpret_cast<uintptr_t>(a->oqs) & 3u) == 0),
              "q36_gdn_prompt: oq must be 16-byte and oqs 4-byte aligned");
  const size_t need = q36_gdn_prompt_workspace_bytes(a->rows, a->B);
  Q36_REQUIRE(a->workspace_bytes >= need, "q36_gdn_prompt: workspace %zu < %zu bytes", a->workspace_bytes, need);
  Q36_REQUIRE((reinterpret_cast<uintptr_t>(a->workspace) & 255u) == 0, "q36_gdn_prompt: workspace must be 256-byte aligned");
  PromptDev d{a->B, a->rows, a->slots, a->idx_i64 & 1, a->dt_f32 ? 1 : 0, a->eps, a->scale,
              static_cast<const uint16_t*>(a->mixed), static_cast<const uint16_t*>(a->z), static_cast<const uint16_t*>(a->a),
              static_cast<const uint16_t*>(a->b), static_cast<uint16_t*>(a->conv_state), a->cs_slot,
              static_cast<const uint16_t*>(a->conv_w), a->A_log, a->dt_bias, a->h0, a->qsl, a->state_idx, a->prefix,
              static_cast<const uint16_t*>(a->norm_w), static_cast<uint16_t*>(a->out), static_cast<uint8_t*>(a->oq), a->oqs};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  prompt_steps_kernel<<<(unsigned)a->B * PHK, 512, 0, st>>>(d);
  return check_launch("q36_gdn_prompt");
}
