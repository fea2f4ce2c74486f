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
    // Phi(x) by Abramowitz & Stegun 7.1.26: for z = |x| / sqrt(2), erfc(z) = (a1 t + ... + a5 t^5) exp(-z^2)
    // with t = 1 / (1 + p z), |error| <= 1.5e-7; its exponential is the one that the density needs
    const float z = fabsf(x) * 0.70710678f;
    const float e = __expf(-z * z), t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, z, 1.f));
    const float q = fmaf(fmaf(fmaf(fmaf(1.061405429f, t, -1.453152027f), t, 1.421413741f), t, -0.284496736f), t,
                         0.254829592f) * t * e * 0.5f;
    const float c = x < 0.f ? q : 1.f - q;
    a = x * c;
    d = fmaf(x * 0.39894228f, e, c);
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

// Three outputs a tile (h, and g and u for training), so its end moves 192 KB: 8192 rows of 768 through
// 2 x 2048 take 80 us (0.64 PFLOP/s; at 128x128 73 by itself, but the whole step 352 against 344),
// 16384 of 2048 through 2 x 5632 680 to 730 us (1.04 to 1.11 PFLOP/s).
template <int ACT>
struct EpiGate {
  u16 *g, *u, *h;  // [N][F8]; g and u null without gradients
  int64_t ld;
  template <int NI, int MI>
  struct Pre {};
  template <int NI, int MI>
  __device__ __forceinline__ void load(const g16::Ctx&, Pre<NI, MI>&) const {}
  template <int NI, int MI>
  __device__ __forceinline__ void run(const g16::Ctx& c, const Pre<NI, MI>&, f32x4 (&acc)[NI][MI]) const {
    constexpr int H = NI / 2;
    const g16::RowStage<H * 16> st{c.stage, c.lane};
    g16::unroll<MI>([&](auto J) {
      constexpr int j = J.value;
      g16::pin(acc, j);
      auto out = [&](u16* o) {
        st.turn();
#pragma unroll
        for (int q = 0; q < st.GETS; ++q) {
          const int m = c.m0 + j * 16 + st.row(q), n = c.n0 + st.col();
          const uint4 v = st.get(q);
          if (m < c.M && n < ld) *reinterpret_cast<uint4*>(o + (int64_t)m * ld + n) = v;
        }
        st.turn();
      };
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const int n = c.n0 + i * 16 + 4 * (c.lane >> 4);
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float a, d;
          act_both<ACT>(acc[i][j][k], a, d);
          v[k] = n + k < c.N ? a * acc[i + H][j][k] : 0.f;  // columns F..F8: zeros for the next product
        }
        st.put(i, pack4bf(v[0], v[1], v[2], v[3]));
      }
      out(h);
      if (g) {
#pragma unroll
        for (int i = 0; i < H; ++i) st.put(i, pack4bf(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]));
        out(g);
#pragma unroll
        for (int i = 0; i < H; ++i)
          st.put(i, pack4bf(acc[i + H][j][0], acc[i + H][j][1], acc[i + H][j][2], acc[i + H][j][3]));
        out(u);
      }
    });
  }
};

__device__ __forceinline__ void unpack4(uint2 q, float (&v)[4]) {
  v[0] = bf2f((u16)q.x);
  v[1] = bf2f((u16)(q.x >> 16));
  v[2] = bf2f((u16)q.y);
  v[3] = bf2f((u16)(q.y >> 16));
}

// g and u come from memory as they went there: whole rows of 16 bytes a lane, turned into the
// accumulators' layout in LDS, and dg and du back. At 128x128, two blocks a CU: four rows of 16-bit values
// read and written per product of K = 768 make it memory's (8192 x 2048 x 768: 60 us, 147 MB at
// 2.4 TB/s; 16384 x 5632 x 2048: 510 to 535 us). The loads of one group of rows run ahead of its use; all of
// a tile's loads ahead of everything was slower (64 and 572 us).
template <int ACT>
struct EpiGateGrad {
  const u16 *g, *u;  // [N][ld]
  u16* dgu;          // [N][2 ld]: dg, then du
  int64_t ld;
  template <int NI, int MI>
  struct Pre {};
  template <int NI, int MI>
  __device__ __forceinline__ void load(const g16::Ctx&, Pre<NI, MI>&) const {}
  template <int NI, int MI>
  __device__ __forceinline__ void run(const g16::Ctx& c, const Pre<NI, MI>&, f32x4 (&acc)[NI][MI]) const {
    const g16::RowStage<NI * 16> st{c.stage, c.lane};
    constexpr int G = st.GETS;
    uint4 gq[G], uq[G];
    auto fetch = [&](int j) {
#pragma unroll
      for (int q = 0; q < G; ++q) {
        const int m = min(c.m0 + j * 16 + st.row(q), c.M - 1);
        const int64_t o = (int64_t)m * ld + min(c.n0 + st.col(), (int)ld - 8);
        gq[q] = *reinterpret_cast<const uint4*>(g + o);
        uq[q] = *reinterpret_cast<const uint4*>(u + o);
      }
    };
    fetch(0);
    g16::unroll<MI>([&](auto J) {
      constexpr int j = J.value;
      g16::pin(acc, j);
      auto turned = [&](const uint4 (&q)[G], uint2 (&r)[NI]) {
#pragma unroll
        for (int k = 0; k < G; ++k) st.set(k, q[k]);
        st.turn();
#pragma unroll
        for (int i = 0; i < NI; ++i) r[i] = st.take(i);
        st.turn();
      };
      uint2 gr[NI], ur[NI];
      turned(gq, gr);
      turned(uq, ur);
      if (j + 1 < MI) fetch(j + 1);
      uint2 du[NI];
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int n = c.n0 + i * 16 + 4 * (c.lane >> 4);
        float gv[4], uv[4], x[4], y[4];
        unpack4(gr[i], gv);
        unpack4(ur[i], uv);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float a, d;
          act_both<ACT>(gv[k], a, d);
          const bool in = n + k < c.N;
          x[k] = in ? acc[i][j][k] * uv[k] * d : 0.f;
          y[k] = in ? acc[i][j][k] * a : 0.f;
        }
        st.put(i, pack4bf(x[0], x[1], x[2], x[3]));
        du[i] = pack4bf(y[0], y[1], y[2], y[3]);
      }
      auto out = [&](u16* o) {
        st.turn();
#pragma unroll
        for (int q = 0; q < G; ++q) {
          const int m = c.m0 + j * 16 + st.row(q), n = c.n0 + st.col();
          const uint4 v = st.get(q);
          if (m < c.M && n < ld) *reinterpret_cast<uint4*>(o + (int64_t)m * 2 * ld + n) = v;
        }
        st.turn();
      };
      out(dgu);
#pragma unroll
      for (int i = 0; i < NI; ++i) st.put(i, du[i]);
      out(dgu + ld);
    });
  }
};

// Few rows (serving): a block of eight waves per 16 columns, each wave an eighth of k, its fragments
// straight from memory: a lane's 16 bytes are eight consecutive k of one weight row, and every weight is
// read once, so LDS would only add a trip. Two launches, each a memory latency or two long: one row of
// 768 through 2048 columns takes 7.9 us in a graph (1.2 TB/s; through the core's tiles, 64 rows high, k cut
// by splits with a third launch, 20 us), of 2048 through 5632 22 us (3.1 TB/s). The rows are read again
// by every block: at 32 rows 13 and 40 us (core: 22 and 48), at 64 rows 18 and 58, so up to 32 come here.
// MB: groups of 16 rows.
constexpr int FEW = 32;
template <int MB, bool DUAL, class Out>
__device__ __forceinline__ void few_rows(const u16* __restrict__ x, int64_t ldx, int N, const u16* __restrict__ w0,
                                         const u16* __restrict__ w1, int64_t ldw, int F, int K, const Out& out) {
  constexpr int W = DUAL ? 2 : 1, D = 4;  // steps of 32 k whose loads are in flight together
  __shared__ float part[8][W][MB * 256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n0 = blockIdx.x * 16, r = lane & 15, kq = 8 * (lane >> 4);
  const int steps = (K + 31) / 32, first = steps * wave / 8, last = steps * (wave + 1) / 8;
  const u16* pw[W];
  pw[0] = w0 + (int64_t)min(n0 + r, F - 1) * ldw;
  if constexpr (DUAL) pw[1] = w1 + (int64_t)min(n0 + r, F - 1) * ldw;
  const u16* px[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) px[b] = x + (int64_t)min(b * 16 + r, N - 1) * ldx;
  f32x4 acc[W][MB];
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int b = 0; b < MB; ++b) acc[i][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = first; s < last; s += D) {
    bf16x8 fw[D][W], fx[D][MB];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      // rows are whole up to the next multiple of 8 past K, zeros there; nothing is read behind that
      const int k = (s + d) * 32 + kq;
      const bool on = s + d < last && k < K;
#pragma unroll
      for (int i = 0; i < W; ++i) fw[d][i] = on ? *reinterpret_cast<const bf16x8*>(pw[i] + k) : bf16x8{};
#pragma unroll
      for (int b = 0; b < MB; ++b) fx[d][b] = on ? *reinterpret_cast<const bf16x8*>(px[b] + k) : bf16x8{};
    }
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
      for (int i = 0; i < W; ++i)
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[i][b] = mfma16(fw[d][i], fx[d][b], acc[i][b]);
  }
  // acc[k]: column n0 + 4 (lane >> 4) + k of row lane & 15
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int b = 0; b < MB; ++b)
      *reinterpret_cast<f32x4*>(&part[wave][i][(b * 16 + r) * 16 + 4 * (lane >> 4)]) = acc[i][b];
  __syncthreads();
  for (int e = threadIdx.x; e < MB * 256; e += 512) {
    float v[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      v[i] = part[0][i][e];
#pragma unroll
      for (int q = 1; q < 8; ++q) v[i] += part[q][i][e];
    }
    if ((e >> 4) < N) out(e >> 4, n0 + (e & 15), v);
  }
}

template <int ACT, int MB>
__global__ void __launch_bounds__(512) ffn_gate_few(const u16* __restrict__ x, int64_t ldx, int N, const u16* __restrict__ wg,
                                                    const u16* __restrict__ wu, int64_t ldw, int F, int F8, int K,
                                                    u16* __restrict__ g, u16* __restrict__ u, u16* __restrict__ h) {
  few_rows<MB, true>(x, ldx, N, wg, wu, ldw, F, K, [&](int m, int n, const float (&v)[2]) {
    if (n >= F8) return;
    const int64_t o = (int64_t)m * F8 + n;
    const bool in = n < F;  // columns F..F8: zeros for the next product
    float a, d;
    act_both<ACT>(v[0], a, d);
    h[o] = in ? f2bf(a * v[1]) : (u16)0;
    if (g) {
      g[o] = in ? f2bf(v[0]) : (u16)0;
      u[o] = in ? f2bf(v[1]) : (u16)0;
    }
  });
}
template <int MB>
__global__ void __launch_bounds__(512) ffn_down_few(const u16* __restrict__ h, int64_t ldh, int N, const u16* __restrict__ w,
                                                    int64_t ldw, int K, int F, u16* __restrict__ y) {
  few_rows<MB, false>(h, ldh, N, w, w, ldw, K, F, [&](int m, int n, const float (&v)[1]) {
    if (n < K) y[(int64_t)m * K + n] = f2bf(v[0]);
  });
}

template <int MB>
void forward_few(const FfnShape& s, const u16* x, int64_t ldx, const FfnWeights& w, int act, u16* g, u16* u, u16* h, u16* y,
                 hipStream_t st) {
  auto gate = [&](auto A) {
    ffn_gate_few<A.value, MB><<<g16::cdiv(s.F8, 16), 512, 0, st>>>(x, ldx, s.N, w.gate, w.up, w.ldgu, s.F, s.F8, s.K, g, u, h);
  };
  switch (act) {
    case ACT_SILU: gate(std::integral_constant<int, ACT_SILU>{}); break;
    case ACT_GELU: gate(std::integral_constant<int, ACT_GELU>{}); break;
    case ACT_GELU_TANH: gate(std::integral_constant<int, ACT_GELU_TANH>{}); break;
    case ACT_RELU: gate(std::integral_constant<int, ACT_RELU>{}); break;
    default: gate(std::integral_constant<int, ACT_SIGMOID>{}); break;
  }
  ffn_down_few<MB><<<g16::cdiv(s.K, 16), 512, 0, st>>>(h, s.F8, s.N, w.down, w.ldd, s.K, s.F, y);
}

g16::Side side(const u16* p, int64_t ld, int ext) {
  g16::Side s;
  s.p[0] = p;
  s.ld = ld;
  s.ext = ext;
  return s;
}

int gate_tile(const FfnShape& s) { return g16::plan(s.N, 2 * (int64_t)s.F, s.K, 1, 1, false, false, 1.5, g16::T_DUAL).tile; }

template <int ACT>
void up_gate(const FfnShape& s, const u16* x, int64_t ldx, const FfnWeights& w, u16* g, u16* u, u16* h, hipStream_t st) {
  g16::Args a;
  a.m = side(x, ldx, s.N);
  a.n = side(w.gate, w.ldgu, s.F);
  a.n.alt = w.up;
  a.M = s.N;
  a.N = s.F;
  a.K = s.K;
  g16::launch<g16::KC, g16::KC, true>(gate_tile(s), a, EpiGate<ACT>{g, u, h, s.F8}, st);
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
  g16::launch_tile<g16::KC, g16::KS, 128, 2, false, 0>(a, g16::Ragged(), EpiGateGrad<ACT>{g, u, dgu, s.F8}, st);
}

}  // namespace

#ifndef MIHVD_F16
FfnPlan ffn_plan(const FfnShape& s) {
  const g16::Plan p[4] = {g16::product_plan(s.N, s.K, s.F), g16::product_plan(s.K, s.F, s.N),
                          g16::product_plan(s.F, s.K, s.N, 1, 2), g16::product_plan(s.N, s.K, s.F, 2)};
  FfnPlan r{s.N <= FEW ? 0 : gate_tile(s), {}, {}};
  for (int i = 0; i < 4; ++i) r.tile[i] = p[i].tile, r.splits[i] = p[i].splits;
  return r;
}
#endif

void ffn_forward_16(const FfnShape& s, const u16* x, int64_t ldx, const FfnWeights& w, int act, u16* g, u16* u, u16* h,
                    u16* y, c10::Device dev, hipStream_t st) {
  if (s.N <= 16) return forward_few<1>(s, x, ldx, w, act, g, u, h, y, st);
  if (s.N <= FEW) return forward_few<2>(s, x, ldx, w, act, g, u, h, y, st);
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
  g16::product<g16::KC, g16::KC>(a, y, nullptr, s.K, dev, st);
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
    g16::product<g16::KS, g16::KS>(a, dwd, nullptr, s.F, dev, st);
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
    g16::product<g16::KS, g16::KS>(a, dwg ? dwg : dwu, dwg ? dwu : nullptr, s.K, dev, st);
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
    g16::product<g16::KC, g16::KS>(a, dx, nullptr, s.K, dev, st);
  }
}

MIHVD_OPNS_END
