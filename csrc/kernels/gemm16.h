// Matrix-product core of the transformer-step operators (linear_ce.hip, gated_ffn.hip,
// newton_schulz.hip): 16-bit operands (bf16, or fp16 in a -DMIHVD_F16 build), fp32 accumulation,
// with the operator's own work in the epilogue.
//
//   out[m][n] = sum over segments s and k < K of  Pm_s(m, k) * Pn_s(n, k)
//
// Each side is stored K-contiguous ("KC", [row][k]) or K-strided ("KS", [k][row]), so no operand is
// ever transposed in memory: forward products are KC x KC, products with a weight along its other
// axis KC x KS, weight gradients KS x KS. Segments concatenate products along k (the two halves of
// a gated input gradient; the three products hi*hi + hi*lo + lo*hi of split fp32 values).
//
// The n side feeds the MFMA's A operand and the m side its B operand, so a lane's four accumulators
// are four consecutive n of one m (v_mfma_f32_16x16x32: C[4*(l>>4)+i][l&15]): packed 8-byte stores
// along the output rows, and a reduction over n stays in the lane but for two exchanges.
//
// Staging is global_load_lds_dwordx4 into double-buffered swizzled LDS images; one barrier per
// 64-wide k tile. Out-of-range rows are clamped to the last row (their products only reach outputs
// that are never stored); k positions past K are read from a page of zeros on both sides.
//
// What a caller guarantees (checked on the host by G16Side makers): 16-byte aligned bases, leading
// dimensions and KS extents that are multiples of 8 elements, KC rows that hold zeros (or any
// finite values against zeros) from K to the next multiple of 8.
#pragma once

#include <ATen/ATen.h>

#include "common.h"

MIHVD_OPNS_BEGIN
namespace g16 {

enum { KC = 0, KS = 1 };
constexpr int BK = 64;

static __device__ __attribute__((aligned(16))) const unsigned zeros16[4] = {0, 0, 0, 0};

struct Side {
  const u16* p[3] = {nullptr, nullptr, nullptr};  // one base per segment
  const u16* alt = nullptr;                       // DUAL: the second matrix of interleaved rows
  int64_t ld = 0;                                 // elements between rows (KC) / between k (KS)
  int64_t bs = 0;                                 // elements between batch entries
  int ext = 0;                                    // rows (KC); storage extent, a multiple of 8 (KS)
};

struct Args {
  Side m, n;
  int M = 0, N = 0, K = 0;  // K: per segment
  int nseg = 1, batch = 1, splits = 1;
  int sym = 0;                  // out is symmetric (M == N): only tiles with nt >= mt run
  const int* dyn_m = nullptr;   // device count that replaces M (tiles past it exit)
  const int* dyn_k = nullptr;   // device count that replaces K
  int tiles_m = 0, tiles_n = 0; // filled by launch()
};

// What an epilogue sees of its wave: the wave's first m and n, and the tile it belongs to.
struct Ctx {
  int m0, n0;      // origin of the wave tile (DUAL: n0 in columns of one matrix)
  int M, N;        // bounds (M after dyn_m)
  int mt, nt;      // tile indices
  int wm, wn;      // wave position in the tile
  int batch, split, lane;
};

// Row permutation of a KS image: 16-byte chunks of k row `k` are XORed with 2*h(k), so that the
// eight k rows a half wave reads with ds_read_b64_tr_b16 land in different 32-byte bank groups.
template <int R>
__device__ __forceinline__ int ks_h(int k) {
  if constexpr (R >= 128) return (k & 3) | (((k >> 3) & 1) << 2);
  else return ((k >> 1) & 1) | (((k >> 3) & 1) << 1);
}

// One side's staging of an [R x 64] (KC) or [64 x R] (KS) tile by NT threads.
template <int LAYOUT, int R, int NT, bool DUAL>
struct Stage {
  static constexpr int J = R * 8 / NT;
  static_assert(J * NT == R * 8 && NT % 64 == 0, "whole chunks per thread");
  uint32_t off[J];

  __device__ __forceinline__ void init(const Side& s, int x0, int t) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int i = t + j * NT;
      if constexpr (LAYOUT == KC) {
        const int row = i >> 3, src = (i & 7) ^ (row & 7);
        const int r = DUAL ? ((row >> 7) << 6) + (row & 63) : row;  // 64 rows of p, 64 of alt, ...
        off[j] = (uint32_t)min(r, s.ext - 1 - x0) * (uint32_t)s.ld * 2u + (uint32_t)src * 16u;
      } else {
        constexpr int RC = R / 8;
        const int k = i / RC, src = (i % RC) ^ (2 * ks_h<R>(k));
        off[j] = (uint32_t)k * (uint32_t)s.ld * 2u + (uint32_t)min(8 * src, s.ext - 8 - x0) * 2u;
      }
    }
  }
  // k of the chunk that thread t stages in its j-th load
  __device__ __forceinline__ static int kpos(int j, int t) {
    const int i = t + j * NT;
    if constexpr (LAYOUT == KC) return 8 * ((i & 7) ^ ((i >> 3) & 7));
    else return i / (R / 8);
  }
  __device__ __forceinline__ static bool is_alt(int j) { return DUAL && (((j * NT) >> 3) & 64); }

  __device__ __forceinline__ void issue(const char* base, const char* alt, u16* lds, int t, int krem) const {
    const int w0 = (t >> 6) * 64;
    if (krem >= BK) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const char* g = (is_alt(j) ? alt : base) + off[j];
        __builtin_amdgcn_global_load_lds((const void*)g, (void __attribute__((address_space(3)))*)(lds + (j * NT + w0) * 8),
                                         16, 0, 0);
      }
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const char* g = (is_alt(j) ? alt : base) + off[j];
        g = kpos(j, t) < krem ? g : (const char*)zeros16;
        __builtin_amdgcn_global_load_lds((const void*)g, (void __attribute__((address_space(3)))*)(lds + (j * NT + w0) * 8),
                                         16, 0, 0);
      }
    }
  }
};

// Fragment of 16 rows from row `row0` (a multiple of 16) of a staged image, k block kk (32 wide).
template <int LAYOUT, int R>
__device__ __forceinline__ bf16x8 frag(const u16* lds, int row0, int kk, int lane) {
  if constexpr (LAYOUT == KC) {
    const int r = row0 + (lane & 15);
    return frag_ld128(lds + r * 64 + 8 * ((kk * 4 + (lane >> 4)) ^ (lane & 7)));
  } else {
    const int k = kk * 32 + 8 * (lane >> 4) + ((lane & 15) >> 2);
    const int chunk = ((row0 >> 3) ^ (2 * ks_h<R>(k))) + ((lane & 3) >> 1);
    const u16* p = lds + k * R + 8 * chunk + 4 * (lane & 1);
    return frag_tr(p, p + 4 * R);
  }
}

// Tile order: the blocks that one XCD runs (every eighth) take a contiguous run of tiles, walked in
// groups of eight m tiles, so that the 32 tiles an XCD has in flight share rows of both operands in
// its L2.
__device__ __forceinline__ void tile_of(const Args& a, int& batch, int& split, int& mt, int& nt) {
  const int nb = gridDim.x, id = blockIdx.x;
  const int q = nb >> 3, r = nb & 7, x = id & 7;
  int pos = x * q + min(x, r) + (id >> 3);
  const int tiles = a.sym ? a.tiles_m * (a.tiles_m + 1) / 2 : a.tiles_m * a.tiles_n;
  batch = pos / (tiles * a.splits);
  pos -= batch * tiles * a.splits;
  split = pos / tiles;
  pos -= split * tiles;
  if (a.sym) {
    mt = 0;
    while (pos >= a.tiles_m - mt) {
      pos -= a.tiles_m - mt;
      ++mt;
    }
    nt = mt + pos;
    return;
  }
  constexpr int G = 8;
  const int g = pos / (G * a.tiles_n), first = g * G;
  const int gs = min(G, a.tiles_m - first);
  pos -= g * G * a.tiles_n;
  mt = first + pos % gs;
  nt = pos / gs;
}

template <int LM, int LN, int TM, int TN, int WM, int WN, bool DUAL, class Epi>
__global__ void __launch_bounds__(64 * WM * WN) gemm16_kernel(const Args a, const Epi epi) {
  constexpr int NT = 64 * WM * WN, WTM = TM / WM, WTN = TN / WN, MI = WTM / 16, NI = WTN / 16;
  __shared__ u16 lds[2][(TM + TN) * BK];
  int batch, split, mt, nt;
  tile_of(a, batch, split, mt, nt);
  const int M = a.dyn_m ? *a.dyn_m : a.M, K = a.dyn_k ? *a.dyn_k : a.K;
  const int x0m = mt * TM, x0n = nt * (DUAL ? TN / 2 : TN);
  if (x0m >= M) return;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int wm = wave % WM, wn = wave / WM;

  Stage<LM, TM, NT, false> sm;
  Stage<LN, TN, NT, DUAL> sn;
  sm.init(a.m, x0m, t);
  sn.init(a.n, x0n, t);
  const int64_t tm0 = a.m.bs * batch + (LM == KC ? (int64_t)x0m * a.m.ld : x0m);
  const int64_t tn0 = a.n.bs * batch + (LN == KC ? (int64_t)x0n * a.n.ld : x0n);
  const int64_t stepm = LM == KC ? BK : BK * a.m.ld, stepn = LN == KC ? BK : BK * a.n.ld;

  const int kiters = (K + BK - 1) / BK, total = kiters * a.nseg;
  const int per = (total + a.splits - 1) / a.splits;
  const int it0 = split * per, it1 = min(total, it0 + per);

  f32x4 acc[NI][MI];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto issue = [&](int it, int buf) {
    const int seg = a.nseg == 1 ? 0 : it / kiters, kp = it - seg * kiters;
    const u16* pm = seg == 0 ? a.m.p[0] : seg == 1 ? a.m.p[1] : a.m.p[2];
    const u16* pn = seg == 0 ? a.n.p[0] : seg == 1 ? a.n.p[1] : a.n.p[2];
    const int krem = K - kp * BK;
    sm.issue((const char*)(pm + tm0 + kp * stepm), nullptr, lds[buf], t, krem);
    sn.issue((const char*)(pn + tn0 + kp * stepn), DUAL ? (const char*)(a.n.alt + tn0 + kp * stepn) : nullptr,
             lds[buf] + TM * BK, t, krem);
  };

  if (it0 < it1) issue(it0, 0);
  for (int it = it0; it < it1; ++it) {
    const int buf = (it - it0) & 1;
    __syncthreads();  // this tile has landed; every wave is done reading the other buffer
    if (it + 1 < it1) issue(it + 1, buf ^ 1);
    const u16* am = lds[buf];
    const u16* an = lds[buf] + TM * BK;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      bf16x8 fb[MI];
#pragma unroll
      for (int j = 0; j < MI; ++j) fb[j] = frag<LM, TM>(am, wm * WTM + j * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        int row;
        if constexpr (DUAL) {
          const int col = wn * (WTN / 2) + (i % (NI / 2)) * 16;
          row = ((col >> 6) << 7) + (i >= NI / 2 ? 64 : 0) + (col & 63);
        } else {
          row = wn * WTN + i * 16;
        }
        const bf16x8 fa = frag<LN, TN>(an, row, kk, lane);
#pragma unroll
        for (int j = 0; j < MI; ++j) acc[i][j] = mfma16(fa, fb[j], acc[i][j]);
      }
    }
  }
  Ctx c;
  c.m0 = x0m + wm * WTM;
  c.n0 = x0n + wn * (DUAL ? WTN / 2 : WTN);
  c.M = M;
  c.N = a.N;
  c.mt = mt;
  c.nt = nt;
  c.wm = wm;
  c.wn = wn;
  c.batch = batch;
  c.split = split;
  c.lane = lane;
  epi.template run<NI, MI>(c, acc);
}

inline int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
inline int64_t up8(int64_t x) { return (x + 7) / 8 * 8; }

template <int LM, int LN, int TM, int TN, int WM, int WN, bool DUAL = false, class Epi>
void launch(Args a, const Epi& e, hipStream_t stream) {
  a.tiles_m = cdiv(a.M, TM);
  a.tiles_n = cdiv(a.N, DUAL ? TN / 2 : TN);
  const int64_t tiles = a.sym ? (int64_t)a.tiles_m * (a.tiles_m + 1) / 2 : (int64_t)a.tiles_m * a.tiles_n;
  const int64_t blocks = tiles * a.splits * a.batch;
  if (blocks <= 0) return;
  gemm16_kernel<LM, LN, TM, TN, WM, WN, DUAL, Epi><<<dim3((unsigned)blocks), dim3(64 * WM * WN), 0, stream>>>(a, e);
}

// ---- epilogue helpers ---------------------------------------------------------------------- //
// Store four consecutive values of a row: one 8-byte store when `vec` (row starts 8-byte aligned).
__device__ __forceinline__ void store4(u16* row, int n, int N, bool vec, float a, float b, float c, float d) {
  if (vec && n + 3 < N) {
    *reinterpret_cast<uint2*>(row + n) = pack4bf(a, b, c, d);
    return;
  }
  if (n < N) row[n] = f2bf(a);
  if (n + 1 < N) row[n + 1] = f2bf(b);
  if (n + 2 < N) row[n + 2] = f2bf(c);
  if (n + 3 < N) row[n + 3] = f2bf(d);
}

// out[batch][m][n] = alpha * acc, rounded once to the 16-bit format; alpha times an optional device
// scalar. `out[]` holds one base per batch entry.
struct EpiStore {
  u16* out[2];
  int64_t ld;
  float alpha;
  const float* dev_alpha;
  template <int NI, int MI>
  __device__ __forceinline__ void run(const Ctx& c, f32x4 (&acc)[NI][MI]) const {
    const float al = dev_alpha ? alpha * *dev_alpha : alpha;
    u16* o = c.batch == 0 ? out[0] : out[1];
    const bool vec = (ld & 3) == 0;
#pragma unroll
    for (int j = 0; j < MI; ++j) {
      const int m = c.m0 + j * 16 + (c.lane & 15);
      if (m >= c.M) continue;
      u16* row = o + (int64_t)m * ld;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int n = c.n0 + i * 16 + 4 * (c.lane >> 4);
        store4(row, n, c.N, vec, acc[i][j][0] * al, acc[i][j][1] * al, acc[i][j][2] * al, acc[i][j][3] * al);
      }
    }
  }
};

// fp32 slab of one k split: slab[batch * splits + split][m][n] (+)= acc. ld is a multiple of 4.
struct EpiSlab {
  float* slab;
  int64_t ld, stride;
  int splits, add;
  template <int NI, int MI>
  __device__ __forceinline__ void run(const Ctx& c, f32x4 (&acc)[NI][MI]) const {
    float* o = slab + (int64_t)(c.batch * splits + c.split) * stride;
#pragma unroll
    for (int j = 0; j < MI; ++j) {
      const int m = c.m0 + j * 16 + (c.lane & 15);
      if (m >= c.M) continue;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int n = c.n0 + i * 16 + 4 * (c.lane >> 4);
        if (n < ld) {
          f32x4* q = reinterpret_cast<f32x4*>(o + (int64_t)m * ld + n);
          *q = add ? *q + acc[i][j] : acc[i][j];
        }
      }
    }
  }
};

// out[batch][m][n] = alpha * sum of the slabs, in split order
static __global__ void __launch_bounds__(256) slab_sum(const float* __restrict__ slab, int splits, int64_t stride,
                                                       int64_t ld, int M, int N, u16* __restrict__ out0,
                                                       u16* __restrict__ out1, int64_t ldo, float alpha,
                                                       const float* __restrict__ dev_alpha) {
  const int n4 = (N + 3) >> 2;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t m = i / n4;
  const int n = (int)(i - m * n4) * 4;
  if (m >= M) return;
  const float al = dev_alpha ? alpha * *dev_alpha : alpha;
  const float* p = slab + (int64_t)blockIdx.y * splits * stride + m * ld + n;
  f32x4 s = *reinterpret_cast<const f32x4*>(p);
  for (int q = 1; q < splits; ++q) s += *reinterpret_cast<const f32x4*>(p + q * stride);
  store4((blockIdx.y ? out1 : out0) + m * ldo, n, N, (ldo & 3) == 0, s[0] * al, s[1] * al, s[2] * al, s[3] * al);
}

// k splits for a product of `tiles` output tiles: enough blocks for every CU, at least four k tiles
// each, so that a slab's round trip through memory stays small against the products it carries.
inline int pick_splits(int64_t tiles, int64_t kiters) {
  const int64_t want = device_cu_count() / std::max<int64_t>(tiles, 1);
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, kiters / 4), 64));
}

// A product rounded once into 16-bit outputs (one or two batch entries), split along k when its
// tiles alone leave CUs idle.
template <int LM, int LN>
void product(Args a, u16* out0, u16* out1, int64_t ldo, float alpha, const float* dev_alpha, c10::Device dev,
             hipStream_t stream) {
  const int64_t tiles = (int64_t)cdiv(a.M, 128) * cdiv(a.N, 128) * a.batch;
  const int64_t kiters = (int64_t)cdiv(a.K, BK) * a.nseg;
  a.splits = pick_splits(tiles, kiters);
  if (a.splits == 1) {
    launch<LM, LN, 128, 128, 2, 2>(a, EpiStore{{out0, out1}, ldo, alpha, dev_alpha}, stream);
    return;
  }
  const int64_t ld = up8(a.N), stride = (int64_t)a.M * ld;
  at::Tensor slab = at::empty({a.batch * a.splits * stride}, at::TensorOptions().device(dev).dtype(at::kFloat));
  launch<LM, LN, 128, 128, 2, 2>(a, EpiSlab{slab.data_ptr<float>(), ld, stride, a.splits, 0}, stream);
  slab_sum<<<dim3(cdiv((int64_t)a.M * ((a.N + 3) / 4), 256), a.batch), 256, 0, stream>>>(
      slab.data_ptr<float>(), a.splits, stride, ld, a.M, a.N, out0, out1, ldo, alpha, dev_alpha);
}

}  // namespace g16
MIHVD_OPNS_END
