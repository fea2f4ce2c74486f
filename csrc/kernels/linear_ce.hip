// Softmax cross entropy of a vocabulary projection, without keeping the logits.
//
//   z = h W^T + b;   L_r = lse_r - z[r][y_r],  lse_r = log sum_v exp(z[r][v])
//   dz = g_r (exp(z - lse) - onehot);  dh = dz W;  dW = dz^T h;  db = sum_r dz
//
// lse is kept as two numbers, the row's maximum and log sum exp(z - max), and the maximum is subtracted before
// anything is scaled or rounded: logits of any size (words masked by -1e30 or the type's lowest value, all words
// of a row masked alike) keep exact differences.
//
// Forward: the logits exist only as MFMA accumulators; every wave reduces its columns of a row to a
// running (max, sum of exp) pair in fp32 and writes that pair, and the row's own label logit where
// it holds it. A second kernel joins the pairs of a row. Backward recomputes the logits piece by
// piece of the vocabulary, writes dz of the piece in 16 bits (the operand format of the two products
// that follow), and multiplies it into dW (that piece's rows, final) and dh (fp32 slabs, summed over
// pieces and k splits in a fixed order). No atomics: results repeat bit for bit.
//
// Rows whose label is `ignore_index` are dropped before anything is multiplied: the labelled rows
// are compacted (their count stays on the device), so a masked-LM head over all positions costs what
// its masked positions cost.
//
// dz is held as (exp(z - lse) - onehot) * (g_r / G) * 2^shift with G = max |g_r|; G and 2^-shift come
// back in the epilogues. bf16 needs no shift; fp16 takes 2^14, so that probabilities down to 4e-9
// stay normal numbers (fp16's smallest is 6e-5) and 1.0 stays far from 65504. With row weights that is a
// probability times g_r / G: dW needs the weights inside its sum over rows, and one 16-bit dz serves both
// products, so in fp16 rows far below the largest weight lose digits of their small probabilities.
#include "gemm16.h"

#include "transformer.h"

MIHVD_OPNS_BEGIN

namespace {
#ifdef MIHVD_F16
constexpr float DZ_SCALE = 16384.f, DZ_LOG2 = 14.f;
#else
constexpr float DZ_SCALE = 1.f, DZ_LOG2 = 0.f;
#endif

// Sum of n over a block of 1024, for every thread.
__device__ __forceinline__ int count_block(int n, int* sh) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = n;
  __syncthreads();
  int tot = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) tot += sh[i];
  return tot;
}

// Labelled rows of each chunk of rows.
__global__ void __launch_bounds__(1024) lce_count(const int64_t* __restrict__ labels, int N, int64_t ignore, int chunk,
                                                  int* __restrict__ counts) {
  __shared__ int sh[16];
  const int64_t r0 = (int64_t)blockIdx.x * chunk, r1 = min((int64_t)N, r0 + chunk);
  int n = 0;
  for (int64_t r = r0 + threadIdx.x; r < r1; r += 1024) n += labels[r] != ignore;
  const int tot = count_block(n, sh);
  if (threadIdx.x == 0) counts[blockIdx.x] = tot;
}

// Compacts the labelled rows: their row numbers, their labels in 32 bits (-1: outside the vocabulary),
// every row's place among them, their count, and their hidden vectors. A block takes 16 rows, a wave
// each, and counts the labels ahead of them by itself: of all rows (up to 16384 of them: 64 KB a block on
// average, out of L2), or of its chunk on top of the chunks' counts. AGAIN: blocks go round, where there are more
// rows than a launch of fewer than 2^32 threads has waves (the loop costs 3 of 7 us at 8192 rows).
constexpr int64_t GATHER_BLOCKS = int64_t(1) << 21;
template <bool AGAIN>
__global__ void __launch_bounds__(1024) lce_gather(const int64_t* __restrict__ labels, int N, int V, int64_t ignore,
                                                   const int* __restrict__ counts, int chunk, const u16* __restrict__ h,
                                                   int64_t s0, int64_t s1, int K, int K8, const LceRowsOut rw,
                                                   u16* __restrict__ out) {
  __shared__ int sh[16], own[16];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  for (int64_t first = (int64_t)blockIdx.x * 16; first < N; first += (int64_t)gridDim.x * 16) {
    int n = 0;
    int64_t from = 0;
    if (counts) {
      const int c = (int)(first / chunk);
      for (int i = t; i < c; i += 1024) n += counts[i];
      from = (int64_t)c * chunk;
    }
    for (int64_t r = from + t; r < first; r += 1024) n += labels[r] != ignore;
    const int64_t r = first + w;
    const int64_t y = r < N ? labels[r] : ignore;
    const bool on = y != ignore;
    if (AGAIN && first != (int64_t)blockIdx.x * 16) __syncthreads();  // own[] and sh[] have been read
    if (lane == 0) own[w] = on;
    int pos = count_block(n, sh);  // its barriers publish own[] too
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < w) pos += own[i];
    if (lane == 0 && r < N) {
      rw.inv[r] = on ? pos : -1;
      if (on) {
        rw.idx[pos] = (int)r;
        rw.label[pos] = y >= 0 && y < V ? (int)y : -1;
      }
      if (r == N - 1) *rw.cnt = pos + (on ? 1 : 0);
      if (r == 0) *rw.done = 0;
    }
    if (on) {
      const u16* src = h + r * s0;
      u16* dst = out + (int64_t)pos * K8;
      if (s1 == 1 && (s0 & 7) == 0 && ((uintptr_t)h & 15) == 0 && K == K8) {
        for (int k = lane * 8; k < K; k += 512) *reinterpret_cast<uint4*>(dst + k) = *reinterpret_cast<const uint4*>(src + k);
      } else {
        for (int k = lane; k < K8; k += 64) dst[k] = k < K ? src[(int64_t)k * s1] : (u16)0;
      }
    }
    if (!AGAIN) return;
  }
}

// A lane's bias values, as its accumulators hold the columns.
template <bool BIAS, int NI>
struct BiasRegs {
  float v[BIAS ? NI : 1][4];
  __device__ __forceinline__ void load(const void* b, int kind, int n0, int N, int lane) {
    if constexpr (BIAS) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int n = min(n0 + i * 16 + 4 * (lane >> 4) + k, N - 1);
          v[i][k] = kind == 1 ? static_cast<const float*>(b)[n] : bf2f(static_cast<const u16*>(b)[n]);
        }
    }
  }
  __device__ __forceinline__ float add(float z, int i, int k) const {
    if constexpr (BIAS) return z + v[i][k];
    else return z;
  }
};

// logits in place; columns past N (only a tile that ends inside has them) become -inf
template <bool BIAS, int NI, int MI>
__device__ __forceinline__ void logits(const g16::Ctx& c, const BiasRegs<BIAS, NI>& b, f32x4 (&acc)[NI][MI], int j,
                                       f32x4 (&z)[NI]) {
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) z[i][k] = b.add(acc[i][j][k], i, k);
  if (c.n0 + NI * 16 > c.N) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c.n0 + i * 16 + 4 * (c.lane >> 4) + k >= c.N) z[i][k] = -INFINITY;
  }
}

// Does column `lab` lie among the lane's? Then (lab - first) >> 4 and & 3 are its i and k.
template <int NI>
__device__ __forceinline__ bool mine(const g16::Ctx& c, int lab, int& d) {
  d = lab - (c.n0 + 4 * (c.lane >> 4));
  return d >= 0 && d < NI * 16 && (d & 15) < 4;
}

// A value with lane ^ 16's and lane ^ 32's joined to it, without a trip through LDS: a swap of two copies
// of v gives every lane the even and the odd rows' (the lower and the upper half's) values.
template <class F>
__device__ __forceinline__ float join_rows(float v, const F& f) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// exp(z - top) 2^c. The difference comes first: z log2(e) and top log2(e), rounded each for itself, would be
// off by 2^-24 of z, which is any number of powers of two where z is a large mask.
constexpr float LOG2E = 1.44269504f;
__device__ __forceinline__ float exp_from(float z, float top) { return __builtin_amdgcn_exp2f((z - top) * LOG2E); }
__device__ __forceinline__ float exp_from(float z, float top, float c) {
  return __builtin_amdgcn_exp2f(fmaf(z - top, LOG2E, c));
}

// Statistics of one wave's columns: part[row][piece] = (max, sum of exp(z - max)), and the label's logit.
// A logit costs a read, half a max, a subtraction, a product, an exponential (as long as four others) and an add:
// about 4 us a
// 256x256 tile behind 17 us of products at K = 768. 1229 x 30522 x 768: 84 us (0.69 PFLOP/s, 600 tiles in
// three rounds on 256 CUs); 8192 x 65536 x 1024: 0.98 to 1.08 ms (1.0 to 1.1 PFLOP/s; at 128x128 1.2 to 1.26).
template <bool BIAS>
struct EpiStats {
  const void* bias;
  int bias_kind;
  const int* label;   // compact labels
  float2* part;       // [rows][npart]
  int npart;
  float* zlab;        // [rows]
  template <int NI, int MI>
  struct Pre {
    BiasRegs<BIAS, NI> b;
    int lab[MI];
  };
  template <int NI, int MI>
  __device__ __forceinline__ void load(const g16::Ctx& c, Pre<NI, MI>& p) const {
    p.b.load(bias, bias_kind, c.n0, c.N, c.lane);
#pragma unroll
    for (int j = 0; j < MI; ++j) p.lab[j] = label[min(c.m0 + j * 16 + (c.lane & 15), c.M - 1)];
  }
  template <int NI, int MI>
  __device__ __forceinline__ void run(const g16::Ctx& c, const Pre<NI, MI>& p, f32x4 (&acc)[NI][MI]) const {
    const int slot = c.nt * 2 + c.wn;  // two waves along a tile's columns
    g16::unroll<MI>([&](auto J) {
      constexpr int j = J.value;
      g16::pin(acc, j);
      const int m = c.m0 + j * 16 + (c.lane & 15);
      f32x4 z[NI];
      logits(c, p.b, acc, j, z);
      int d;
      if (mine<NI>(c, p.lab[j], d) && m < c.M) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (d == i * 16 + k) zlab[m] = z[i][k];
      }
      float mx = z[0][0];
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) mx = fmaxf(mx, z[i][k]);
      mx = join_rows(mx, [](float a, float b) { return fmaxf(a, b); });
      const float ref = mx == -INFINITY ? 0.f : mx;  // a strip of -inf adds nothing, without inf - inf
      f32x4 s4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) s4[k] += exp_from(z[i][k], ref);
      float s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
      s = join_rows(s, [](float a, float b) { return a + b; });
      if (c.lane < 16 && m < c.M) part[(int64_t)m * npart + slot] = make_float2(mx, s);
    });
  }
};

// Joins the pairs of every row: WPR waves a row, four where there are few rows, so that their loads are in
// flight together. Writes lse (compact: maximum, log of the sum) and the row's loss (all rows), and into `out`, if
// given, their sum
// or mean: every block adds up its rows, and the block that ends last adds up the blocks, both in a fixed
// order.
template <int WPR>
__global__ void __launch_bounds__(256) lce_finish(const float2* __restrict__ part, int npart,
                                                  const float* __restrict__ zlab, const int* __restrict__ label,
                                                  const int* __restrict__ inv, int N, int V, float2* __restrict__ lse,
                                                  float* __restrict__ rows, float* __restrict__ blocks,
                                                  int* __restrict__ done, const int* __restrict__ cnt, int mean,
                                                  float* __restrict__ out) {
  constexpr int RPB = 4 / WPR;
  __shared__ float2 sh[4];
  __shared__ int last;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = wave % WPR;
  float total = 0.f;
  const int n = out ? *cnt : N;
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < n; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t r = r0 + wave / WPR;
    const int c = r >= n ? -1 : out ? (int)r : inv[r];
    float mx = -INFINITY, s = 0.f;
    if (c >= 0) {
      const float2* q = part + (int64_t)c * npart;
      auto join = [&](const float2 v) {
        const float top = fmaxf(mx, v.x), ref = top == -INFINITY ? 0.f : top;
        s = s * __expf(mx - ref) + v.y * __expf(v.x - ref);
        mx = top;
      };
      int p = sub * 64 + lane;
      for (; p + 3 * WPR * 64 < npart; p += 4 * WPR * 64) {  // four loads in flight
        float2 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = q[p + k * WPR * 64];
#pragma unroll
        for (int k = 0; k < 4; ++k) join(v[k]);
      }
      for (; p < npart; p += WPR * 64) join(q[p]);
      const float all = wave_max(mx), ref = all == -INFINITY ? 0.f : all;
      s = wave_sum(s * __expf(mx - ref));
      mx = all;
    }
    if constexpr (WPR > 1) {
      if (lane == 0) sh[wave] = make_float2(mx, s);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < WPR; ++i) mx = fmaxf(mx, sh[i].x);
      const float ref = mx == -INFINITY ? 0.f : mx;
      s = 0.f;
#pragma unroll
      for (int i = 0; i < WPR; ++i) s += sh[i].y * __expf(sh[i].x - ref);
      __syncthreads();
    }
    if (lane == 0 && sub == 0 && r < n) {
      float v = 0.f;
      if (c >= 0) {
        const int y = label[c];
        // a label outside the vocabulary has no loss: NaN, and NaN gradients through lse
        const bool in = y >= 0 && y < V;
        const float2 l = in ? make_float2(mx, logf(s)) : make_float2(NAN, NAN);
        lse[c] = l;
        v = (l.x - (in ? zlab[c] : 0.f)) + l.y;
      }
      if (out) total += v;
      else rows[r] = v;
    }
  }
  if (!out) return;
  if (lane == 0) sh[wave].x = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = 0.f;
    for (int i = 0; i < 4; ++i) t += sh[i].x;
    __hip_atomic_store(blocks + blockIdx.x, t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = __hip_atomic_fetch_add(done, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  float t = 0.f;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += 256)
    t += __hip_atomic_load(blocks + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  t = wave_sum(t);
  __syncthreads();
  if (lane == 0) sh[wave].x = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    float tot = 0.f;
    for (int i = 0; i < 4; ++i) tot += sh[i].x;
    *out = mean ? tot / (float)*cnt : tot;
  }
}

// (1229 x 30522 x 768 with a bias at 128x128: 86 us; a piece of 32768 of 8192 x 65536 x 1024 at 256x256:
// 560 to 600 us, 0.92 to 0.98 PFLOP/s, 0.54 GB of it written.)
// dz of one piece of the vocabulary (its columns start at v0), times DZ_SCALE, and with BIAS its sums over
// the wave's rows (the bias gradient's terms). ROWS: rows have weights of their own. The scale is
// folded into the exponent; the label's column is put right afterwards, by the one lane that has it.
template <bool BIAS, bool ROWS>
struct EpiDz {
  const void* bias;  // from v0 on
  int bias_kind;
  const int* label;
  const float2* lse;      // maximum, log of the sum
  const float* rowscale;  // g_r / G per compact row
  int v0;
  u16* dz;                // [rows][ld]
  int64_t ld;
  float* dbp;             // [m waves][ld]
  template <int NI, int MI>
  struct Pre {
    BiasRegs<BIAS, NI> b;
    int lab[MI];
    float2 ls[MI];
    float rs[ROWS ? MI : 1];
  };
  template <int NI, int MI>
  __device__ __forceinline__ void load(const g16::Ctx& c, Pre<NI, MI>& p) const {
    p.b.load(bias, bias_kind, c.n0, c.N, c.lane);
#pragma unroll
    for (int j = 0; j < MI; ++j) {
      const int m = min(c.m0 + j * 16 + (c.lane & 15), c.M - 1);
      p.lab[j] = label[m];
      p.ls[j] = lse[m];
      if constexpr (ROWS) p.rs[j] = rowscale[m];
    }
  }
  template <int NI, int MI>
  __device__ __forceinline__ void run(const g16::Ctx& c, const Pre<NI, MI>& p, f32x4 (&acc)[NI][MI]) const {
    f32x4 sum[BIAS ? NI : 1];
#pragma unroll
    for (int i = 0; i < (BIAS ? NI : 1); ++i) sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const g16::RowStage<NI * 16> st{c.stage, c.lane};
    g16::unroll<MI>([&](auto J) {
      constexpr int j = J.value;
      g16::pin(acc, j);
      const int m = c.m0 + j * 16 + (c.lane & 15);
      const float top = p.ls[j].x, sub = DZ_LOG2 - p.ls[j].y * LOG2E;
      f32x4 z[NI];
      logits(c, p.b, acc, j, z);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) z[i][k] = exp_from(z[i][k], top, sub);
      int d;
      if (mine<NI>(c, p.lab[j] - v0, d)) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (d == i * 16 + k && c.n0 + i * 16 + 4 * (c.lane >> 4) + k < c.N) z[i][k] -= DZ_SCALE;
      }
      if constexpr (ROWS) {
#pragma unroll
        for (int i = 0; i < NI; ++i) z[i] *= p.rs[j];
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        if constexpr (BIAS) {
          if (m < c.M) sum[i] += z[i];
        }
        st.put(i, pack4bf(z[i][0], z[i][1], z[i][2], z[i][3]));
      }
      st.turn();
#pragma unroll
      for (int g = 0; g < st.GETS; ++g) {
        const int r = c.m0 + j * 16 + st.row(g), n = c.n0 + st.col();
        const uint4 v = st.get(g);
        if (r < c.M && n < ld)  // columns N..ld are the zeros that the next products read
          *reinterpret_cast<uint4*>(dz + (int64_t)r * ld + n) = v;
      }
      st.turn();
    });
    if constexpr (BIAS) {
      float* o = dbp + (int64_t)(c.mt * 2 + c.wm) * ld;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int n = c.n0 + i * 16 + 4 * (c.lane >> 4);
        f32x4 t = sum[i];
#pragma unroll
        for (int k = 0; k < 4; ++k) t[k] = row_sum16(t[k]);
        if ((c.lane & 15) == 0 && n < ld) *reinterpret_cast<f32x4*>(o + n) = t;
      }
    }
  }
};

// The ends of the two gradients that are summed up: blocks below `dh_blocks` write dh of every row, the sum of
// its slabs or zeros where the label was ignored; the others db of a piece of the vocabulary. (Past GRAD_BLOCKS,
// which with db's blocks stay below 2^32 threads, dh's blocks go round again.)
constexpr int64_t GRAD_BLOCKS = int64_t(1) << 23;
__global__ void __launch_bounds__(256) lce_grads(int dh_blocks, const float* __restrict__ slab,
                                                 const int* __restrict__ splits, int64_t ld, const int* __restrict__ inv, int N, int K,
                                                 u16* __restrict__ dh, const float* __restrict__ dbp, int64_t ldb, int tm,
                                                 int V, void* __restrict__ db, int kind, const int* __restrict__ cnt,
                                                 const LceGrad g) {
  const float scale = g16::scalar(g.scale, g.div) * (1.f / DZ_SCALE);
  const int rows = *cnt;
  if ((int)blockIdx.x < dh_blocks) {
    const int nslab = *splits;
    const int k4 = (K + 3) / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)N * k4; i += (int64_t)dh_blocks * 256) {
      const int64_t r = i / k4;
      const int k = (int)(i - r * k4) * 4;
      const int c = inv[r];
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
      if (c >= 0) {
        const int64_t stride = (int64_t)rows * ld;
        const float* p = slab + (int64_t)c * ld + k;
        int q = 0;
        for (; q + 8 <= nslab; q += 8) {  // eight loads in flight
          f32x4 v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = *reinterpret_cast<const f32x4*>(p + (q + e) * stride);
#pragma unroll
          for (int e = 0; e < 8; ++e) s += v[e];
        }
        for (; q < nslab; ++q) s += *reinterpret_cast<const f32x4*>(p + q * stride);
        s *= scale;
      }
      g16::store4(dh + r * K, k, K, (K & 3) == 0, s[0], s[1], s[2], s[3]);
    }
    return;
  }
  const int64_t v = (int64_t)(blockIdx.x - dh_blocks) * 256 + threadIdx.x;
  if (v >= V) return;
  const int n = (rows + tm - 1) / tm * 2;  // two waves along a tile's rows
  float s = 0.f;
  for (int i = 0; i < n; ++i) s += dbp[(int64_t)i * ldb + v];
  s *= scale;
  if (kind == 1) static_cast<float*>(db)[v] = s;
  else static_cast<u16*>(db)[v] = f2bf(s);
}

template <bool BIAS, class Epi>
void dz_launch(int tile, const g16::Args& a, const Epi& e, hipStream_t st) {
  if constexpr (BIAS) g16::launch_small<g16::KC, g16::KC>(tile, a, e, st);
  else g16::launch<g16::KC, g16::KC>(tile, a, e, st);
}

}  // namespace

#ifndef MIHVD_F16
void lce_plan(LceShape& s) {
  s.tile = g16::plan(s.N, s.V, s.K, 1, 1, false, false, 1.5).tile;
  s.npart = g16::cdiv(s.V, s.tile) * 2;
}
void lce_plan_backward(LceShape& s, LceScratch& x, bool bias) {
  // the bias gradient's sums on top of the accumulators spill at 256x256 (135 us a piece against 84
  // without them, at 1229 x 30522 x 768); at 128x128 they fit
  x.dz_tile = g16::plan(s.N, std::min(x.piece, s.V), s.K, 1, 1, false, false, 1.5, bias ? g16::T_SMALL : g16::T_ALL).tile;
  const g16::Plan p = g16::plan(s.N, s.K, x.piece, 1, 1, false, true);
  x.dh_tile = p.tile;
  x.splits = p.splits;
  x.slab_rows = (int64_t)g16::split_rule(s.N, s.K, x.piece, p, nullptr).cap * p.tile;
  x.dw_tile = g16::plan(std::min(x.piece, s.V), s.K, s.N, 1, 1, false, false).tile;
}
#endif

void lce_forward_16(const LceShape& s, const int64_t* labels, int64_t ignore, const LceRowsOut& rw, const u16* h,
                    int64_t hs0, int64_t hs1, const u16* w, int64_t ldw, const void* bias, int bias_kind, u16* hc,
                    float2* part, float* zlab, float2* lse, float* rows, float* blocks, float* loss, int mean,
                    hipStream_t st) {
  if (s.chunk) lce_count<<<g16::cdiv(s.N, s.chunk), 1024, 0, st>>>(labels, s.N, ignore, s.chunk, rw.counts);
  const int64_t blocks16 = g16::cdiv(s.N, 16);
  auto gather = [&](auto kernel) {
    kernel<<<(int)std::min(blocks16, GATHER_BLOCKS), 1024, 0, st>>>(labels, s.N, s.V, ignore, s.chunk ? rw.counts : nullptr,
                                                                   s.chunk, h, hs0, hs1, s.K, s.K8, rw, hc);
  };
  if (blocks16 <= GATHER_BLOCKS) gather(lce_gather<false>);
  else gather(lce_gather<true>);
  g16::Args a;
  a.m.p[0] = hc;
  a.m.ld = s.K8;
  a.m.ext = s.N;
  a.n.p[0] = w;
  a.n.ld = ldw;
  a.n.ext = s.V;
  a.M = s.N;
  a.N = s.V;
  a.K = s.K;
  a.dyn_m = rw.cnt;
  if (bias) g16::launch<g16::KC, g16::KC>(s.tile, a, EpiStats<true>{bias, bias_kind, rw.label, part, s.npart, zlab}, st);
  else g16::launch<g16::KC, g16::KC>(s.tile, a, EpiStats<false>{nullptr, 0, rw.label, part, s.npart, zlab}, st);
  auto finish = [&](auto kernel, int grid) {
    kernel<<<grid, 256, 0, st>>>(part, s.npart, zlab, rw.label, rw.inv, s.N, s.V, lse, rows, blocks, rw.done, rw.cnt, mean,
                                 loss);
  };
  if (s.N <= LCE_BLOCKS) finish(lce_finish<4>, s.N);
  else finish(lce_finish<1>, std::min(g16::cdiv(s.N, 4), loss ? LCE_BLOCKS : 4096));
}

void lce_backward_16(const LceShape& s, const LceRows& rw, const LceGrad& g, const u16* hc, const u16* w, int64_t ldw,
                     const void* bias, int bias_kind, const float2* lse, const LceScratch& x, u16* dh, u16* dw, void* db,
                     hipStream_t st) {
  // The slabs of all pieces add up, so one rule serves them all: as many splits as suit the labelled rows, which are
  // often few among all (with the head over 8192 positions, 1229 of them labelled, 138 us with the
  // splits that suit 8192 rows).
  const g16::SplitRule rule = g16::split_rule(s.N, s.K, x.piece, {x.dh_tile, x.splits}, x.chosen);
  for (int v0 = 0, first = 1; v0 < s.V; v0 += x.piece, first = 0) {
    const int nv = std::min(x.piece, s.V - v0);
    const u16* wp = w + (int64_t)v0 * ldw;
    {
      g16::Args a;
      a.m.p[0] = hc;
      a.m.ld = s.K8;
      a.m.ext = s.N;
      a.n.p[0] = wp;
      a.n.ld = ldw;
      a.n.ext = nv;
      a.M = s.N;
      a.N = nv;
      a.K = s.K;
      a.dyn_m = rw.cnt;
      const void* b = bias ? static_cast<const char*>(bias) + (int64_t)v0 * (bias_kind == 1 ? 4 : 2) : nullptr;
      auto go = [&](auto B, auto R) {
        EpiDz<B.value, R.value> e{b, bias_kind, rw.label, lse, g.rowscale, v0, x.dz, x.ldz, x.dbp};
        dz_launch<B.value>(x.dz_tile, a, e, st);
      };
      if (bias && g.rowscale) go(std::true_type{}, std::true_type{});
      else if (bias) go(std::true_type{}, std::false_type{});
      else if (g.rowscale) go(std::false_type{}, std::true_type{});
      else go(std::false_type{}, std::false_type{});
    }
    if (dw) {
      g16::Args a;
      a.m.p[0] = x.dz;
      a.m.ld = x.ldz;
      a.m.ext = (int)g16::up8(nv);
      a.n.p[0] = hc;
      a.n.ld = s.K8;
      a.n.ext = s.K8;
      a.M = nv;
      a.N = s.K;
      a.K = s.N;
      a.dyn_k = rw.cnt;
      g16::EpiStore e{{dw + (int64_t)v0 * s.K, nullptr}, s.K, 1.f / DZ_SCALE, g.scale, g.div};
      g16::launch<g16::KS, g16::KS>(x.dw_tile, a, e, st);
    }
    if (dh) {
      g16::Args a;
      a.m.p[0] = x.dz;
      a.m.ld = x.ldz;
      a.m.ext = s.N;
      a.n.p[0] = wp;
      a.n.ld = ldw;
      a.n.ext = s.K8;
      a.M = s.N;
      a.N = s.K;
      a.K = nv;
      a.splits = 64;  // as many as the rule can choose: every slot gets a block
      a.dyn_m = rw.cnt;
      a.rule = rule;
      g16::EpiSlab e{x.slab, s.K8, 0, 1, first ? 0 : 1};
      g16::launch<g16::KC, g16::KS>(x.dh_tile, a, e, st);
    }
    // the pieces' slabs add up: dh is whole behind the last one
    const int dh_blocks = dh && v0 + nv == s.V ? (int)std::min<int64_t>(((int64_t)s.N * ((s.K + 3) / 4) + 255) / 256, GRAD_BLOCKS) : 0;
    const int db_blocks = db ? g16::cdiv(nv, 256) : 0;
    void* dbv = db ? static_cast<char*>(db) + (int64_t)v0 * (bias_kind == 1 ? 4 : 2) : nullptr;
    if (dh_blocks + db_blocks)
      lce_grads<<<dh_blocks + db_blocks, 256, 0, st>>>(dh_blocks, x.slab, x.chosen, s.K8, rw.inv, s.N, s.K, dh, x.dbp, x.ldz,
                                                       x.dz_tile, nv, dbv, bias_kind, rw.cnt, g);
  }
}

MIHVD_OPNS_END
