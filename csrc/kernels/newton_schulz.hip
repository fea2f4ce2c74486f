// Orthogonalising a matrix by Newton-Schulz steps, and the weight update made of it.
//
//   X = u / (|u|_F + eps);   per step  A = X X^T,  B = b A + c A A,  X <- a X + B X
// (for more rows than columns the same on the other side: A = X^T X, X <- a X + X B).
//
// X, A and B are bounded (singular values stay below ~1.3), so they are held in fp16 scaled by 2^12:
// the MFMA rate of bf16 with three more bits. fp32 values are held as two fp16 planes hi + lo (22
// bits) and multiplied as hi hi + hi lo + lo hi, three k segments of one product; the dropped lo lo
// is below 2^-22. A and B are symmetric: only tiles on and above the diagonal are computed, and
// stored twice.
//
// Elements below 2^-26 of the norm lose relative precision in the scaled planes (fp16's smallest
// step is 2^-24); their absolute error is 2^-37, below the fp32 rounding of the sums they enter.
#define MIHVD_F16 1
#include "gemm16.h"

#include "transformer.h"

namespace mihvd {

using namespace f16;

namespace {

constexpr float S = 4096.f, INV_S = 1.f / 4096.f;

struct NsTable {
  const void* src[NS_MAX];
  float* mom[NS_MAX];
};
struct NsOut {
  void* dst[NS_MAX];
};

__device__ __forceinline__ float load_src(const void* p, int kind, int64_t i) {
  if (kind == 0) return static_cast<const float*>(p)[i];
  const u16 h = static_cast<const u16*>(p)[i];
  return kind == 1 ? __uint_as_float((uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
}

// Sum of squares of each matrix, NS_PART partial sums; for Muon the momentum is updated on the way:
// m = mu m + g, u = g + mu m (nesterov) or m.
__global__ void __launch_bounds__(256) ns_norm(const NsTable t, int64_t n, int kind, int muon, float mu, int nesterov,
                                               float* __restrict__ partial) {
  __shared__ float sh[4];
  const int b = blockIdx.y;
  float s = 0.f;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float v = load_src(t.src[b], kind, i);
    if (muon) {
      const float m = fmaf(mu, t.mom[b][i], v);
      t.mom[b][i] = m;
      v = nesterov ? fmaf(mu, m, v) : m;
    }
    s = fmaf(v, v, s);
  }
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) partial[b * NS_PART + blockIdx.x] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// planes of S * v: hi, and lo = the rest
__device__ __forceinline__ void put_planes(u16* p, int64_t plane, int planes, float v) {
  const u16 hi = f2bf(v);
  p[0] = hi;
  if (planes == 2) p[plane] = f2bf(v - bf2f(hi));
}

__global__ void __launch_bounds__(256) ns_scale(const NsTable t, int rows, int cols, int rp, int cp, int planes, int kind,
                                                int muon, float mu, int nesterov, float eps,
                                                const float* __restrict__ partial, u16* __restrict__ x) {
  const int b = blockIdx.y, lane = threadIdx.x & 63;
  const float norm = sqrtf(wave_sum(partial[b * NS_PART + lane]));
  const float inv = S / (norm + eps);
  const int64_t plane = (int64_t)rp * cp;
  u16* o = x + (int64_t)b * planes * plane;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < plane; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / cp;
    const int c = (int)(i - r * cp);
    float v = 0.f;
    if (r < rows && c < cols) {
      const int64_t k = r * cols + c;
      v = load_src(t.src[b], kind, k);
      if (muon) {
        const float m = t.mom[b][k];
        v = nesterov ? fmaf(mu, m, v) : m;
      }
      v *= inv;
    }
    put_planes(o + i, plane, planes, v);
  }
}

// out planes [batch][planes][rows][ld] = alpha * acc + beta * in (planes of the same layout); symmetric
// ones off the diagonal are stored a second time with rows and columns exchanged. N is a multiple of 64.
template <bool IN>
struct EpiPlanes {
  u16* out;
  const u16* in;
  int64_t ld, plane;
  int planes, sym;
  float alpha, beta;
  template <int NI, int MI>
  struct Pre {};
  template <int NI, int MI>
  __device__ __forceinline__ void load(const g16::Ctx&, Pre<NI, MI>&) const {}
  template <int NI, int MI>
  __device__ __forceinline__ void run(const g16::Ctx& c, const Pre<NI, MI>&, f32x4 (&acc)[NI][MI]) const {
    u16* o = out + (int64_t)c.batch * planes * plane;
    const u16* q = IN ? in + (int64_t)c.batch * planes * plane : nullptr;
    const g16::RowStage<NI * 16> st{c.stage, c.lane};
    constexpr int G = st.GETS;
    uint4 iq[2][G];
    auto fetch = [&](int j) {
#pragma unroll
      for (int r = 0; r < G; ++r) {
        const int64_t at = (int64_t)min(c.m0 + j * 16 + st.row(r), c.M - 1) * ld + min(c.n0 + st.col(), c.N - 8);
        iq[0][r] = *reinterpret_cast<const uint4*>(q + at);
        if (planes == 2) iq[1][r] = *reinterpret_cast<const uint4*>(q + plane + at);
      }
    };
    if constexpr (IN) fetch(0);
    g16::unroll<MI>([&](auto J) {
      constexpr int j = J.value;
      g16::pin(acc, j);
      auto write = [&](u16* p) {
        st.turn();
#pragma unroll
        for (int r = 0; r < G; ++r) {
          const int m = c.m0 + j * 16 + st.row(r), n = c.n0 + st.col();
          const uint4 v = st.get(r);
          if (m < c.M && n < c.N) *reinterpret_cast<uint4*>(p + (int64_t)m * ld + n) = v;
        }
        st.turn();
      };
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[i][j] *= alpha;
      if constexpr (IN) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          if (p == 1 && planes == 1) break;
#pragma unroll
          for (int r = 0; r < G; ++r) st.set(r, iq[p][r]);
          st.turn();
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            const uint2 w = st.take(i);
            acc[i][j][0] = fmaf(beta, bf2f((u16)w.x), acc[i][j][0]);
            acc[i][j][1] = fmaf(beta, bf2f((u16)(w.x >> 16)), acc[i][j][1]);
            acc[i][j][2] = fmaf(beta, bf2f((u16)w.y), acc[i][j][2]);
            acc[i][j][3] = fmaf(beta, bf2f((u16)(w.y >> 16)), acc[i][j][3]);
          }
          st.turn();
        }
        if (j + 1 < MI) fetch(j + 1);
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) st.put(i, pack4bf(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]));
      write(o);
      if (planes == 2) {
#pragma unroll
        for (int i = 0; i < NI; ++i) st.put(i, pack4bf(rest(acc[i][j][0]), rest(acc[i][j][1]), rest(acc[i][j][2]), rest(acc[i][j][3])));
        write(o + plane);
      }
      if constexpr (NI * MI > 16) g16::pin(acc, j);  // (kept for the mirror image)
    });
    if (!sym || c.nt == c.mt) return;
    // the mirror image, by blocks of 16 of its rows (this tile's columns)
    constexpr int RS = MI * 16 + 8, CH = MI * 2, GT = 16 * CH / 64;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        if (p == 1 && planes == 1) break;
#pragma unroll
        for (int j = 0; j < MI; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            c.stage[(4 * (c.lane >> 4) + k) * RS + j * 16 + (c.lane & 15)] = f2bf(p ? rest(acc[i][j][k]) : acc[i][j][k]);
        st.turn();
#pragma unroll
        for (int r = 0; r < GT; ++r) {
          const int row = c.lane / CH + r * (64 / CH), col = (c.lane % CH) * 8;
          const int n = c.n0 + i * 16 + row, m = c.m0 + col;
          const uint4 v = *reinterpret_cast<const uint4*>(c.stage + row * RS + col);
          if (n < c.N && m < c.M) *reinterpret_cast<uint4*>(o + p * plane + (int64_t)n * ld + m) = v;
        }
        st.turn();
      }
  }
  __device__ __forceinline__ static float rest(float v) { return v - bf2f(f2bf(v)); }
};

// The last step: v = alpha * acc + beta * X, unscaled, into the result (KIND 0 fp32, 1 bf16, 2 fp16) or the
// weight (3: w = w * decay - step * v).
template <int KIND>
struct EpiFinal {
  NsOut out;
  const u16* in;
  int64_t ld, plane;
  int planes, rows, cols;
  float alpha, beta, decay, step;
  template <int NI, int MI>
  struct Pre {};
  template <int NI, int MI>
  __device__ __forceinline__ void load(const g16::Ctx&, Pre<NI, MI>&) const {}
  template <int NI, int MI>
  __device__ __forceinline__ void run(const g16::Ctx& c, const Pre<NI, MI>&, f32x4 (&acc)[NI][MI]) const {
    const u16* q = in + (int64_t)c.batch * planes * plane;
    void* o = out.dst[c.batch];
    const bool vec = cols % 4 == 0;
    g16::unroll<MI>([&](auto J) {
      constexpr int j = J.value;
      g16::pin(acc, j);
      const int m = c.m0 + j * 16 + (c.lane & 15);
      if (m >= rows) return;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int n = c.n0 + i * 16 + 4 * (c.lane >> 4);
        if (n >= cols) continue;
        const uint2 h = *reinterpret_cast<const uint2*>(q + (int64_t)m * ld + n);
        uint2 l = make_uint2(0, 0);
        if (planes == 2) l = *reinterpret_cast<const uint2*>(q + plane + (int64_t)m * ld + n);
        const float x[4] = {bf2f((u16)h.x) + bf2f((u16)l.x), bf2f((u16)(h.x >> 16)) + bf2f((u16)(l.x >> 16)),
                            bf2f((u16)h.y) + bf2f((u16)l.y), bf2f((u16)(h.y >> 16)) + bf2f((u16)(l.y >> 16))};
        f32x4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = fmaf(beta, x[k], alpha * acc[i][j][k]);
        const int64_t at = (int64_t)m * cols + n;
        if constexpr (KIND == 0 || KIND == 3) {
          float* w = static_cast<float*>(o) + at;
          if (vec && ((uintptr_t)o & 15) == 0) {
            f32x4 r = v;
            if constexpr (KIND == 3) r = *reinterpret_cast<f32x4*>(w) * decay - v * step;
            *reinterpret_cast<f32x4*>(w) = r;
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (n + k < cols) w[k] = KIND == 3 ? fmaf(-step, v[k], w[k] * decay) : v[k];
          }
        } else {
          u16* w = static_cast<u16*>(o) + at;
          u16 r[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) r[k] = KIND == 1 ? __builtin_bit_cast(u16, (__bf16)v[k]) : f2bf(v[k]);
          if (vec && ((uintptr_t)o & 7) == 0) {
            *reinterpret_cast<uint2*>(w) = make_uint2((uint32_t)r[0] | ((uint32_t)r[1] << 16), (uint32_t)r[2] | ((uint32_t)r[3] << 16));
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (n + k < cols) w[k] = r[k];
          }
        }
      }
    });
  }
};

// steps == 0: the normalised matrix itself
__global__ void __launch_bounds__(256) ns_copy_out(const u16* __restrict__ x, const NsOut out, int rows, int cols, int rp,
                                                   int cp, int planes, int kind, int muon, float decay, float step) {
  const int b = blockIdx.y;
  const int64_t plane = (int64_t)rp * cp, n = (int64_t)rows * cols;
  const u16* q = x + (int64_t)b * planes * plane;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / cols, at = r * cp + (i - r * cols);
    float v = bf2f(q[at]);
    if (planes == 2) v += bf2f(q[plane + at]);
    v *= INV_S;
    if (muon) {
      float* w = static_cast<float*>(out.dst[b]) + i;
      *w = fmaf(-step, v, *w * decay);
    } else if (kind == 0) {
      static_cast<float*>(out.dst[b])[i] = v;
    } else if (kind == 1) {
      static_cast<u16*>(out.dst[b])[i] = __builtin_bit_cast(u16, (__bf16)v);
    } else {
      static_cast<u16*>(out.dst[b])[i] = f2bf(v);
    }
  }
}

g16::Side plane_side(const u16* x, int64_t ld, int ext, int64_t plane, int planes, bool second) {
  // segments hi hi, hi lo, lo hi
  g16::Side s;
  s.p[0] = x;
  s.p[1] = second ? x + plane : x;
  s.p[2] = second ? x : x + plane;
  s.ld = ld;
  s.bs = planes * plane;
  s.ext = ext;
  return s;
}

}  // namespace

void ns_run(const NsGroup& g, const NsParams& p, const NsScratch& sc, hipStream_t st) {
  using namespace g16;
  NsTable tab;
  NsOut out;
  for (int i = 0; i < NS_MAX; ++i) {
    tab.src[i] = g.src[i];
    tab.mom[i] = g.mom[i];
    out.dst[i] = g.dst[i];
  }
  const int64_t n = (int64_t)g.rows * g.cols, px = (int64_t)g.rp * g.cp, pa = (int64_t)g.sp * g.sp;
  const int grid = (int)std::min<int64_t>(512, (px + 255) / 256);
  ns_norm<<<dim3(NS_PART, g.count), 256, 0, st>>>(tab, n, p.src_kind, p.muon, p.momentum, p.nesterov, sc.partial);
  ns_scale<<<dim3(grid, g.count), 256, 0, st>>>(tab, g.rows, g.cols, g.rp, g.cp, g.planes, p.src_kind, p.muon, p.momentum,
                                               p.nesterov, p.eps, sc.partial, sc.x0);
  const float step = p.lr * p.scale;
  if (p.steps == 0) {
    ns_copy_out<<<dim3(grid, g.count), 256, 0, st>>>(sc.x0, out, g.rows, g.cols, g.rp, g.cp, g.planes, p.src_kind, p.muon,
                                                     p.decay, step);
    return;
  }
  // All sides are padded to 64 with zeros, which the products keep: a zero row or column of X gives zero
  // rows and columns of A, B and the next X.
  const bool tall = g.rp > g.cp;
  const int nseg = g.planes == 2 ? 3 : 1;
  const int big = std::max(g.rp, g.cp);
  const int t_gram = plan(g.sp, g.sp, big, nseg, g.count, true, false).tile;
  const int t_poly = plan(g.sp, g.sp, g.sp, nseg, g.count, true, false).tile;
  const int t_upd = plan(g.rp, g.cp, g.sp, nseg, g.count, false, false).tile;
  u16 *x = sc.x0, *y = sc.x1;
  for (int it = 0; it < p.steps; ++it) {
    Args a;
    a.batch = g.count;
    a.nseg = nseg;
    a.sym = 1;
    a.M = a.N = g.sp;
    a.K = big;
    const Side xk = plane_side(x, g.cp, g.rp, px, g.planes, false);       // rows of X
    const Side xk2 = plane_side(x, g.cp, g.rp, px, g.planes, true);
    const Side xs = plane_side(x, g.cp, g.cp, px, g.planes, false);       // columns of X
    const Side xs2 = plane_side(x, g.cp, g.cp, px, g.planes, true);
    const EpiPlanes<false> gram{sc.gram, nullptr, g.sp, pa, g.planes, 1, INV_S, 0.f};
    a.m = tall ? xs : xk;
    a.n = tall ? xs2 : xk2;
    if (tall) launch<KS, KS>(t_gram, a, gram, st);
    else launch<KC, KC>(t_gram, a, gram, st);
    a.K = g.sp;
    a.m = plane_side(sc.gram, g.sp, g.sp, pa, g.planes, false);
    a.n = plane_side(sc.gram, g.sp, g.sp, pa, g.planes, true);
    launch<KC, KC>(t_poly, a, EpiPlanes<true>{sc.poly, sc.gram, g.sp, pa, g.planes, 1, p.c * INV_S, p.b}, st);
    a.sym = 0;
    a.M = g.rp;
    a.N = g.cp;
    // tall: X B, rows of X against rows of the symmetric B; else B X
    a.m = tall ? xk : plane_side(sc.poly, g.sp, g.sp, pa, g.planes, false);
    a.n = tall ? plane_side(sc.poly, g.sp, g.sp, pa, g.planes, true) : xs2;
    if (it + 1 < p.steps) {
      const EpiPlanes<true> upd{y, x, g.cp, px, g.planes, 0, INV_S, p.a};
      if (tall) launch<KC, KC>(t_upd, a, upd, st);
      else launch<KC, KS>(t_upd, a, upd, st);
    } else {
      auto fin = [&](auto KIND) {
        const EpiFinal<KIND.value> e{out, x, g.cp, px, g.planes, g.rows, g.cols, INV_S * INV_S, p.a * INV_S, p.decay, step};
        if (tall) launch<KC, KC>(t_upd, a, e, st);
        else launch<KC, KS>(t_upd, a, e, st);
      };
      if (p.muon) fin(std::integral_constant<int, 3>{});
      else if (p.src_kind == 0) fin(std::integral_constant<int, 0>{});
      else if (p.src_kind == 1) fin(std::integral_constant<int, 1>{});
      else fin(std::integral_constant<int, 2>{});
    }
    std::swap(x, y);
  }
}

}  // namespace mihvd
