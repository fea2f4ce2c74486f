// Orthogonalising a matrix by Newton-Schulz steps, and the weight update made of it.
//
//   X = u / (|u|_F + eps);   per step  A = X X^T,  B = a I + b A + c A A,  X <- B X
// (a X + (b A + c A A) X with the first term inside the product: X is read once a step, and B's entries
// get smaller, hence their rounding: near singular values of one its diagonal is 0.7, not -2.7)
// with the smaller side of the matrix as X's rows (a tall one is turned on the way in and out), so that
// matrices of different lengths, wide or tall, run in one batch wherever their smaller sides agree.
//
// X, A and B are bounded (singular values stay below ~1.3), so they are held in fp16 scaled by 2^12:
// the MFMA rate of bf16 with three more bits. fp32 values are held as two fp16 planes hi + lo (22
// bits) and multiplied as hi hi + hi lo + lo hi in one pass over both planes; the dropped lo lo is below
// 2^-22. A and B are symmetric: only tiles on and above the diagonal are computed, and
// stored twice.
//
// The matrices of six layers of 768 (40 M elements, fp32) take 2.5 ms for five steps, of which
// 5 x 150 us are X X^T, 5 x 75 us B, 4 x 240 us and 310 us X <- B X (0.79 PFLOP/s of the three products;
// one block a CU, as the four planes' two buffers fill the LDS, whose reads and copies take as long as the
// MFMAs), and 2 x 94 us the norm and the scaled planes (5.1 TB/s).
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

template <int KIND>
__device__ __forceinline__ float load_src(const void* p, int64_t i) {
  if constexpr (KIND == 0) return static_cast<const float*>(p)[i];
  const u16 h = static_cast<const u16*>(p)[i];
  return KIND == 1 ? __uint_as_float((uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
}
// four consecutive values (the caller has checked the alignment)
template <int KIND>
__device__ __forceinline__ f32x4 load4(const void* p, int64_t i) {
  if constexpr (KIND == 0) {
    return *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const u16*>(p) + i);
    const u16 h[4] = {(u16)w.x, (u16)(w.x >> 16), (u16)w.y, (u16)(w.y >> 16)};
    f32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = KIND == 1 ? __uint_as_float((uint32_t)h[k] << 16) : (float)__builtin_bit_cast(_Float16, h[k]);
    return v;
  }
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// Sum of squares of each matrix, NS_PART partial sums; for Muon the momentum is updated on the way:
// m = mu m + g, u = g + mu m (nesterov) or m. Bound by memory: one read of each input, one write of m. In 64
// bits: the squares of fp32 values above 2^64 or below 2^-75 leave fp32's range.
template <int KIND>
__global__ void __launch_bounds__(256) ns_norm(const NsGroup t, int muon, float mu, int nesterov, double* __restrict__ partial) {
  __shared__ double sh[4];
  const NsMat& q = t.m[blockIdx.y];
  const int64_t n = (int64_t)q.rows * q.cols, stride = (int64_t)gridDim.x * 1024;
  const bool vec = n % 4 == 0 && ((uintptr_t)q.src & (KIND ? 7 : 15)) == 0 && (!muon || ((uintptr_t)q.mom & 15) == 0);
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  if (vec) {
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += stride) {
      f32x4 v = load4<KIND>(q.src, i);
      if (muon) {
        f32x4 m = *reinterpret_cast<f32x4*>(q.mom + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          m[k] = fmaf(mu, m[k], v[k]);
          v[k] = nesterov ? fmaf(mu, m[k], v[k]) : m[k];
        }
        *reinterpret_cast<f32x4*>(q.mom + i) = m;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] = fma((double)v[k], (double)v[k], s[k]);
    }
  } else {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += stride / 4) {
      float v = load_src<KIND>(q.src, i);
      if (muon) {
        const float m = fmaf(mu, q.mom[i], v);
        q.mom[i] = m;
        v = nesterov ? fmaf(mu, m, v) : m;
      }
      s[0] = fma((double)v, (double)v, s[0]);
    }
  }
  const double w = wave_sum64((s[0] + s[1]) + (s[2] + s[3]));
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = w;
  __syncthreads();
  if (threadIdx.x == 0) partial[blockIdx.y * NS_PART + blockIdx.x] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// X = S u / (|u| + eps) into planes, with the smaller side as rows: a 64 x 64 tile a block, turned in LDS
// where the matrix is tall; zeros in the padding.
template <int KIND>
__global__ void __launch_bounds__(256) ns_scale(const NsGroup t, int muon, float mu, int nesterov, float eps,
                                                const double* __restrict__ partial, u16* __restrict__ x) {
  __shared__ float sh[64][65];
  const NsMat& q = t.m[blockIdx.y];
  const int tl = q.len / 64, tiles = t.side / 64 * tl;
  const double inv = S / (sqrt(wave_sum64(partial[blockIdx.y * NS_PART + (threadIdx.x & 63)])) + eps);
  const bool tall = q.rows > q.cols;
  const int64_t plane = (int64_t)t.side * q.len;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int ts = tile / tl * 64, tn = tile % tl * 64;  // along the side, along the length
    const int r0 = tall ? tn : ts, c0 = tall ? ts : tn;
    const bool vec = q.cols % 4 == 0 && ((uintptr_t)q.src & (KIND ? 7 : 15)) == 0 && (!muon || ((uintptr_t)q.mom & 15) == 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = threadIdx.x / 16 + i * 16, c = (threadIdx.x & 15) * 4;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (r0 + r < q.rows) {
        const int64_t at = (int64_t)(r0 + r) * q.cols + c0 + c;
        if (vec && c0 + c < q.cols) {
          v = load4<KIND>(q.src, at);
          if (muon) {
            const f32x4 m = *reinterpret_cast<const f32x4*>(q.mom + at);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = nesterov ? fmaf(mu, m[k], v[k]) : m[k];
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (c0 + c + k < q.cols) {
              v[k] = load_src<KIND>(q.src, at + k);
              if (muon) v[k] = nesterov ? fmaf(mu, q.mom[at + k], v[k]) : q.mom[at + k];
            }
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) sh[r][c + k] = (float)(v[k] * inv);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = threadIdx.x / 8 + i * 32, c = (threadIdx.x & 7) * 8;
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = tall ? sh[c + k][r] : sh[r][c + k];
      u16* o = x + q.off + (int64_t)(ts + r) * q.len + tn + c;
      const uint2 h0 = pack4bf(v[0], v[1], v[2], v[3]), h1 = pack4bf(v[4], v[5], v[6], v[7]);
      *reinterpret_cast<uint4*>(o) = make_uint4(h0.x, h0.y, h1.x, h1.y);
      if (t.planes == 2) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] -= bf2f(f2bf(v[k]));
        const uint2 l0 = pack4bf(v[0], v[1], v[2], v[3]), l1 = pack4bf(v[4], v[5], v[6], v[7]);
        *reinterpret_cast<uint4*>(o + plane) = make_uint4(l0.x, l0.y, l1.x, l1.y);
      }
    }
    __syncthreads();
  }
}

// out planes [batch][planes][rows][ld] = alpha * acc (+ beta * in + diag on the diagonal, `in` being planes of
// the same layout); symmetric ones off the diagonal are stored a second time with rows and columns exchanged. N is a multiple of 64.
template <bool IN>
struct EpiPlanes {
  u16* out;
  const u16* in;
  int64_t ld_, plane_;  // 0: a ragged batch's
  int planes, sym;
  float alpha, beta, diag;
  template <int NI, int MI>
  struct Pre {};
  template <int NI, int MI>
  __device__ __forceinline__ void load(const g16::Ctx&, Pre<NI, MI>&) const {}
  template <int NI, int MI>
  __device__ __forceinline__ void run(const g16::Ctx& c, const Pre<NI, MI>&, f32x4 (&acc)[NI][MI]) const {
    const int64_t ld = ld_ ? ld_ : c.len, plane = ld_ ? plane_ : (int64_t)c.M * c.len;
    const int64_t first = ld_ ? (int64_t)c.batch * planes * plane : c.off;
    u16* o = out + first;
    const u16* q = IN ? in + first : nullptr;
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
        const int d = c.m0 + j * 16 + (c.lane & 15) - c.n0 - 4 * (c.lane >> 4);  // the diagonal's column here
        if (d >= 0 && d < NI * 16 && (d & 15) < 4) {
#pragma unroll
          for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (d == i * 16 + k) acc[i][j][k] += diag;
        }
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

// The last step: v = alpha * acc, unscaled, into the result (KIND 0 fp32, 1 bf16, 2 fp16) or the weight
// (3: w = w * decay - step * v). Column n of X is a row of a tall matrix: those are turned in LDS, eight
// at a time, so that both kinds write whole rows.
struct NsOut {
  void* dst[NS_MAX];
  int rows[NS_MAX], cols[NS_MAX];
  float step[NS_MAX];
};
template <int KIND>
__device__ __forceinline__ void put_out(void* o, int64_t at, float v, float decay, float step) {
  if constexpr (KIND == 3) {
    float* w = static_cast<float*>(o) + at;
    *w = fmaf(-step, v, *w * decay);
  } else if constexpr (KIND == 0) {
    static_cast<float*>(o)[at] = v;
  } else {
    static_cast<u16*>(o)[at] = KIND == 1 ? __builtin_bit_cast(u16, (__bf16)v) : f2bf(v);
  }
}
// four in a row, of which `n` exist
template <int KIND>
__device__ __forceinline__ void put4(void* o, int64_t at, f32x4 v, int n, bool vec, float decay, float step) {
  if (vec && n >= 4) {
    if constexpr (KIND == 0 || KIND == 3) {
      f32x4* w = reinterpret_cast<f32x4*>(static_cast<float*>(o) + at);
      if constexpr (KIND == 3) {
        const f32x4 r = *w;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = fmaf(-step, v[k], r[k] * decay);
      }
      *w = v;
    } else {
      uint32_t r[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) r[k] = KIND == 1 ? __builtin_bit_cast(u16, (__bf16)v[k]) : f2bf(v[k]);
      *reinterpret_cast<uint2*>(static_cast<u16*>(o) + at) = make_uint2(r[0] | (r[1] << 16), r[2] | (r[3] << 16));
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < n) put_out<KIND>(o, at + k, v[k], decay, step);
}
template <int KIND>
struct EpiFinal {
  NsOut out;
  float alpha, decay;
  template <int NI, int MI>
  struct Pre {};
  template <int NI, int MI>
  __device__ __forceinline__ void load(const g16::Ctx&, Pre<NI, MI>&) const {}
  template <int NI, int MI>
  __device__ __forceinline__ void run(const g16::Ctx& c, const Pre<NI, MI>&, f32x4 (&acc)[NI][MI]) const {
    void* o = out.dst[c.batch];
    const int rows = out.rows[c.batch], cols = out.cols[c.batch];
    const float step = out.step[c.batch];
    const bool vec = cols % 4 == 0 && ((uintptr_t)o & 15) == 0;
    if (rows <= cols) {
      g16::unroll<MI>([&](auto J) {
        constexpr int j = J.value;
        g16::pin(acc, j);
        const int m = c.m0 + j * 16 + (c.lane & 15);
        if (m >= rows) return;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int n = c.n0 + i * 16 + 4 * (c.lane >> 4);
          put4<KIND>(o, (int64_t)m * cols + n, acc[i][j] * alpha, cols - n, vec, decay, step);
        }
      });
      return;
    }
    constexpr int RS = MI * 16 + 4, CH = MI * 4, GT = 8 * CH / 64;  // floats a row, float4 a row, float4 a lane
    static_assert(8 * RS * 4 <= 16 * (NI * 16 + 8) * 2, "the stage holds eight rows");
    float* sh = reinterpret_cast<float*>(c.stage);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int j = 0; j < MI; ++j)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            sh[((c.lane >> 4) * 2 + k) * RS + j * 16 + (c.lane & 15)] = acc[i][j][half * 2 + k] * alpha;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int g = 0; g < GT; ++g) {
          const int q = c.lane + g * 64, r = q / CH, m = (q % CH) * 4;
          const f32x4 v = *reinterpret_cast<const f32x4*>(sh + r * RS + m);
          const int n = c.n0 + i * 16 + (r >> 1) * 4 + half * 2 + (r & 1);
          if (n < rows) put4<KIND>(o, (int64_t)n * cols + c.m0 + m, v, cols - c.m0 - m, vec, decay, step);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
  }
};

// no steps: the normalised matrix itself
template <int KIND>
__global__ void __launch_bounds__(256) ns_copy_out(const NsGroup t, const u16* __restrict__ x, const NsOut out, float decay) {
  const NsMat& q = t.m[blockIdx.y];
  const int64_t plane = (int64_t)t.side * q.len, n = (int64_t)q.rows * q.cols;
  const bool tall = q.rows > q.cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / q.cols, c = i - r * q.cols, at = q.off + (tall ? c * q.len + r : r * q.len + c);
    float v = bf2f(x[at]);
    if (t.planes == 2) v += bf2f(x[plane + at]);
    put_out<KIND>(out.dst[blockIdx.y], i, v * INV_S, decay, out.step[blockIdx.y]);
  }
}

g16::Side square_side(const u16* x, int64_t side, int planes) {
  g16::Side s;
  s.p[0] = x;
  s.p[1] = x + side * side;
  s.ld = side;
  s.bs = planes * side * side;
  s.ext = (int)side;
  return s;
}
g16::Side ragged_side(const u16* x, int side) {
  g16::Side s;
  s.p[0] = x;
  s.ext = side;
  return s;
}

// one product: fp16 (tiles by `plan`) or split (by `plan_split`)
template <int LM, int LN, int RAG, bool SMALL, class Epi>
void run_product(int planes, int tile, const g16::Args& a, const Epi& e, hipStream_t st, const g16::Ragged& rg) {
  if (planes == 2) g16::launch_split<LM, LN, RAG>(tile, a, e, st, rg);
  else if constexpr (SMALL) g16::launch_small<LM, LN, RAG>(tile, a, e, st, rg);
  else g16::launch<LM, LN, false, RAG>(tile, a, e, st, rg);
}

template <class F>
void with_kind(const NsParams& p, F&& f) {
  if (p.src_kind == 0) f(std::integral_constant<int, 0>{});
  else if (p.src_kind == 1) f(std::integral_constant<int, 1>{});
  else f(std::integral_constant<int, 2>{});
}

}  // namespace

// Tiles of the three products of a step; the last one of all has its own epilogue, hence a fourth.
NsPlan ns_plan(const NsGroup& g) {
  using namespace g16;
  const int64_t sp = g.side;
  int64_t total = 0;
  for (int i = 0; i < g.count; ++i) total += g.m[i].len;
  auto half = [&](int t) { return (int64_t)cdiv(sp, t) * (cdiv(sp, t) + 1) / 2 * g.count; };  // tiles of a symmetric product
  auto full = [&](int t) {
    int64_t n = 0;
    for (int i = 0; i < g.count; ++i) n += (int64_t)cdiv(sp, t) * cdiv(g.m[i].len, t);
    return n;
  };
  if (g.planes == 2) {
    const int upd = plan_split(full(128), full(64), sp);
    return {plan_split(half(128), half(64), total / g.count), plan_split(half(128), half(64), sp), upd, upd};
  }
  return {plan(sp, sp, total / g.count, 1, g.count, true, false).tile, plan(sp, sp, sp, 1, g.count, true, false, 1.0, T_SMALL).tile,
          plan(sp, total, sp, 1, 1, false, false).tile, plan(sp, total, sp, 1, 1, false, false, 1.0, T_SMALL).tile};
}

void ns_run(const NsGroup& g, const NsParams& p, const NsScratch& sc, hipStream_t st) {
  using namespace g16;
  NsOut out{};
  Ragged rg;
  rg.rows = g.side;
  rg.count = g.count;
  int64_t most = 0;
  for (int i = 0; i < g.count; ++i) {
    out.dst[i] = g.m[i].dst;
    out.rows[i] = g.m[i].rows;
    out.cols[i] = g.m[i].cols;
    out.step[i] = g.m[i].step;
    rg.len[i] = g.m[i].len;
    rg.off[i] = g.m[i].off;
    most = std::max<int64_t>(most, g.m[i].len);
  }
  const int grid = (int)std::min<int64_t>(2048, g.side / 64 * (most / 64));
  with_kind(p, [&](auto K) {
    ns_norm<K.value><<<dim3(NS_PART, g.count), 256, 0, st>>>(g, p.muon, p.momentum, p.nesterov, sc.partial);
    ns_scale<K.value><<<dim3(grid, g.count), 256, 0, st>>>(g, p.muon, p.momentum, p.nesterov, p.eps, sc.partial, sc.x0);
    if (p.steps == 0) {
      if (p.muon) ns_copy_out<3><<<dim3(grid, g.count), 256, 0, st>>>(g, sc.x0, out, p.decay);
      else ns_copy_out<K.value><<<dim3(grid, g.count), 256, 0, st>>>(g, sc.x0, out, p.decay);
    }
  });
  // The sides are padded to 64 with zeros, which the products keep: a zero row or column of X gives zero
  // rows and columns of A, B and the next X.
  const int64_t sp = g.side, pa = sp * sp;
  const NsPlan tile = ns_plan(g);
  u16 *x = sc.x0, *y = sc.x1;
  for (int it = 0; it < p.steps; ++it) {
    Args a;
    a.batch = g.count;
    a.sym = 1;
    a.M = a.N = g.side;
    a.m = a.n = ragged_side(x, g.side);
    run_product<KC, KC, 1, false>(g.planes, tile.gram, a, EpiPlanes<false>{sc.gram, nullptr, sp, pa, g.planes, 1, INV_S, 0.f, 0.f},
                                  st, rg);
    a.K = g.side;
    a.m = a.n = square_side(sc.gram, sp, g.planes);
    run_product<KC, KC, 0, true>(g.planes, tile.poly, a,
                                 EpiPlanes<true>{sc.poly, sc.gram, sp, pa, g.planes, 1, p.c * INV_S, p.b, p.a * S}, st, rg);
    a.sym = 0;
    a.m = square_side(sc.poly, sp, g.planes);
    a.n = ragged_side(x, 0);
    if (it + 1 < p.steps) {
      run_product<KC, KS, 2, false>(g.planes, tile.update, a, EpiPlanes<false>{y, nullptr, 0, 0, g.planes, 0, INV_S, 0.f, 0.f}, st, rg);
    } else {
      auto fin = [&](auto K) {
        run_product<KC, KS, 2, true>(g.planes, tile.last, a, EpiFinal<K.value>{out, INV_S * INV_S, p.decay}, st, rg);
      };
      if (p.muon) fin(std::integral_constant<int, 3>{});
      else with_kind(p, fin);
    }
    std::swap(x, y);
  }
}

}  // namespace mihvd
