// Gated feed-forward block: y = (act(x Wg^T) * (x Wu^T)) Wd^T, and its backward pass.
//
// Forward, first product: one tile holds 64-row groups of Wg and Wu side by side along n, laid out so
// that a lane's accumulators hold gate and up of the same (token, column): the activation and the
// product happen on fp32 accumulators, and only h (and, for training, g and u) reach memory.
// Backward: the product dh = dy Wd never reaches memory either; its epilogue reads g and u and
// writes dg = dh u act'(g) and du = dh act(g) next to each other, which then feed
//   dx = [dg | du] [Wg; Wu]  (two segments of one k loop),  [dWg; dWu] = [dg | du]^T x  (a batch of
//   two),  dWd = dy^T h.
//
// g, u, h, dg and du are rounded to the 16-bit format: they are operands of the next product or of
// act', where half a step of rounding is what the operand format costs anyway.
#include "gemm16.h"

#include "transformer.h"

MIHVD_OPNS_BEGIN

namespace {

__device__ __forceinline__ float sigmoid_f(float x) { return __builtin_amdgcn_rcpf(1.f + __expf(-x)); }

// a = act(x), d = act'(x)
template <int ACT>
__device__ __forceinline__ void act_both(float x, float& a, float& d) {
  if constexpr (ACT == ACT_SILU) {
    const float s = sigmoid_f(x);
    a = x * s;
    d = s * (1.f + x * (1.f - s));
  } else if constexpr (ACT == ACT_GELU) {
    const float c = 0.5f * (1.f + erff(x * 0.70710678f));
    a = x * c;
    d = c + x * 0.39894228f * __expf(-0.5f * x * x);
  } else if constexpr (ACT == ACT_GELU_TANH) {
    // 0.5 (1 + tanh(q)) = sigmoid(2 q)
    const float q = 0.79788456f * (x + 0.044715f * x * x * x);
    const float s = sigmoid_f(2.f * q);
    a = x * s;
    d = s + x * 2.f * s * (1.f - s) * 0.79788456f * (1.f + 0.134145f * x * x);
  } else if constexpr (ACT == ACT_RELU) {
    a = x > 0.f ? x : (x != x ? x : 0.f);
    d = x > 0.f ? 1.f : 0.f;
  } else {
    const float s = sigmoid_f(x);
    a = s;
    d = s * (1.f - s);
  }
}

template <int ACT>
struct EpiGate {
  u16 *g, *u, *h;  // [N][F8]; g and u null without gradients
  int64_t ld;
  template <int NI, int MI>
  __device__ __forceinline__ void run(const g16::Ctx& c, f32x4 (&acc)[NI][MI]) const {
    constexpr int H = NI / 2;
#pragma unroll
    for (int j = 0; j < MI; ++j) {
      const int m = c.m0 + j * 16 + (c.lane & 15);
      if (m >= c.M) continue;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const int n = c.n0 + i * 16 + 4 * (c.lane >> 4);
        if (n >= ld) continue;
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float a, d;
          act_both<ACT>(acc[i][j][k], a, d);
          v[k] = n + k < c.N ? a * acc[i + H][j][k] : 0.f;  // columns F..F8: zeros for the next product
        }
        const int64_t o = (int64_t)m * ld + n;
        *reinterpret_cast<uint2*>(h + o) = pack4bf(v[0], v[1], v[2], v[3]);
        if (g) {
          *reinterpret_cast<uint2*>(g + o) = pack4bf(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
          *reinterpret_cast<uint2*>(u + o) = pack4bf(acc[i + H][j][0], acc[i + H][j][1], acc[i + H][j][2], acc[i + H][j][3]);
        }
      }
    }
  }
};

template <int ACT>
struct EpiGateGrad {
  const u16 *g, *u;  // [N][ld]
  u16* dgu;          // [N][2 ld]: dg, then du
  int64_t ld;
  template <int NI, int MI>
  __device__ __forceinline__ void run(const g16::Ctx& c, f32x4 (&acc)[NI][MI]) const {
#pragma unroll
    for (int j = 0; j < MI; ++j) {
      const int m = c.m0 + j * 16 + (c.lane & 15);
      if (m >= c.M) continue;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int n = c.n0 + i * 16 + 4 * (c.lane >> 4);
        if (n >= ld) continue;
        const int64_t o = (int64_t)m * ld + n;
        const uint2 gq = *reinterpret_cast<const uint2*>(g + o), uq = *reinterpret_cast<const uint2*>(u + o);
        const float gv[4] = {bf2f((u16)gq.x), bf2f((u16)(gq.x >> 16)), bf2f((u16)gq.y), bf2f((u16)(gq.y >> 16))};
        const float uv[4] = {bf2f((u16)uq.x), bf2f((u16)(uq.x >> 16)), bf2f((u16)uq.y), bf2f((u16)(uq.y >> 16))};
        float dg[4], du[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float a, d;
          act_both<ACT>(gv[k], a, d);
          const bool in = n + k < c.N;
          dg[k] = in ? acc[i][j][k] * uv[k] * d : 0.f;
          du[k] = in ? acc[i][j][k] * a : 0.f;
        }
        u16* q = dgu + (int64_t)m * 2 * ld + n;
        *reinterpret_cast<uint2*>(q) = pack4bf(dg[0], dg[1], dg[2], dg[3]);
        *reinterpret_cast<uint2*>(q + ld) = pack4bf(du[0], du[1], du[2], du[3]);
      }
    }
  }
};

g16::Side side(const u16* p, int64_t ld, int ext) {
  g16::Side s;
  s.p[0] = p;
  s.ld = ld;
  s.ext = ext;
  return s;
}

template <int ACT>
void up_gate(const FfnShape& s, const u16* x, int64_t ldx, const FfnWeights& w, u16* g, u16* u, u16* h, hipStream_t st) {
  g16::Args a;
  a.m = side(x, ldx, s.N);
  a.n = side(w.gate, w.ldgu, s.F);
  a.n.alt = w.up;
  a.M = s.N;
  a.N = s.F;
  a.K = s.K;
  g16::launch<g16::KC, g16::KC, true>(g16::plan(s.N, 2 * (int64_t)s.F, s.K, 1, 1, false, false).tile, a, EpiGate<ACT>{g, u, h, s.F8}, st);
}

template <int ACT>
void grad_gate(const FfnShape& s, const u16* dy, int64_t lddy, const FfnWeights& w, const u16* g, const u16* u, u16* dgu,
               hipStream_t st) {
  g16::Args a;
  a.m = side(dy, lddy, s.N);
  a.n = side(w.down, w.ldd, s.F8);
  a.M = s.N;
  a.N = s.F;
  a.K = s.K;
  g16::launch<g16::KC, g16::KS>(g16::plan(s.N, s.F, s.K, 1, 1, false, false).tile, a, EpiGateGrad<ACT>{g, u, dgu, s.F8}, st);
}

}  // namespace

void ffn_forward_16(const FfnShape& s, const u16* x, int64_t ldx, const FfnWeights& w, int act, u16* g, u16* u, u16* h,
                    u16* y, c10::Device dev, hipStream_t st) {
  switch (act) {
    case ACT_SILU: up_gate<ACT_SILU>(s, x, ldx, w, g, u, h, st); break;
    case ACT_GELU: up_gate<ACT_GELU>(s, x, ldx, w, g, u, h, st); break;
    case ACT_GELU_TANH: up_gate<ACT_GELU_TANH>(s, x, ldx, w, g, u, h, st); break;
    case ACT_RELU: up_gate<ACT_RELU>(s, x, ldx, w, g, u, h, st); break;
    default: up_gate<ACT_SIGMOID>(s, x, ldx, w, g, u, h, st); break;
  }
  g16::Args a;
  a.m = side(h, s.F8, s.N);
  a.n = side(w.down, w.ldd, s.K);
  a.M = s.N;
  a.N = s.K;
  a.K = s.F;
  g16::product<g16::KC, g16::KC>(a, y, nullptr, s.K, 1.f, nullptr, dev, st);
}

void ffn_backward_16(const FfnShape& s, const u16* dy, int64_t lddy, const u16* x, int64_t ldx, const FfnWeights& w,
                     int act, const u16* g, const u16* u, const u16* h, u16* dgu, u16* dx, u16* dwg, u16* dwu, u16* dwd,
                     c10::Device dev, hipStream_t st) {
  if (dx || dwg || dwu) {
    switch (act) {
      case ACT_SILU: grad_gate<ACT_SILU>(s, dy, lddy, w, g, u, dgu, st); break;
      case ACT_GELU: grad_gate<ACT_GELU>(s, dy, lddy, w, g, u, dgu, st); break;
      case ACT_GELU_TANH: grad_gate<ACT_GELU_TANH>(s, dy, lddy, w, g, u, dgu, st); break;
      case ACT_RELU: grad_gate<ACT_RELU>(s, dy, lddy, w, g, u, dgu, st); break;
      default: grad_gate<ACT_SIGMOID>(s, dy, lddy, w, g, u, dgu, st); break;
    }
  }
  if (dwd) {
    g16::Args a;
    a.m = side(dy, lddy, s.K8);
    a.n = side(h, s.F8, s.F8);
    a.M = s.K;
    a.N = s.F;
    a.K = s.N;
    g16::product<g16::KS, g16::KS>(a, dwd, nullptr, s.F, 1.f, nullptr, dev, st);
  }
  if (dwg || dwu) {
    g16::Args a;
    a.m = side(dwg ? dgu : dgu + s.F8, 2 * (int64_t)s.F8, s.F8);
    a.m.bs = s.F8;
    a.n = side(x, ldx, s.K8);
    a.M = s.F;
    a.N = s.K;
    a.K = s.N;
    a.batch = dwg && dwu ? 2 : 1;
    g16::product<g16::KS, g16::KS>(a, dwg ? dwg : dwu, dwg ? dwu : nullptr, s.K, 1.f, nullptr, dev, st);
  }
  if (dx) {
    g16::Args a;
    a.m = side(dgu, 2 * (int64_t)s.F8, s.N);
    a.m.p[1] = dgu + s.F8;
    a.n = side(w.gate, w.ldgu, s.K8);
    a.n.p[1] = w.up;
    a.nseg = 2;
    a.M = s.N;
    a.N = s.K;
    a.K = s.F;
    g16::product<g16::KC, g16::KS>(a, dx, nullptr, s.K, 1.f, nullptr, dev, st);
  }
}

MIHVD_OPNS_END
