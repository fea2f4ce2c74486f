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
// Staging is global_load_lds_dwordx4 into double-buffered swizzled LDS images. Out-of-range rows are clamped to the last row (their products only reach outputs
// that are never stored); k positions past K are read from a page of zeros on both sides.
//
// What a caller guarantees (checked on the host by G16Side makers): 16-byte aligned bases, leading
// dimensions and KS extents that are multiples of 8 elements, KC rows that hold zeros (or any
// finite values against zeros) from K to the next multiple of 8.
#pragma once

#include <ATen/ATen.h>

#include <type_traits>

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
  int nseg = 1, batch = 1, splits = 1;  // three segments need K % 64 == 0
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

// Direct global -> LDS copies of 16 bytes a lane (lane l's land at lds + 16 l; lds is wave-uniform).
// Written in asm because the compiler, which cannot tell the two LDS buffers apart, waits for every
// copy in flight before any LDS read; the kernel's own s_waitcnt before the barrier is the wait these
// need. They have no destination registers, and later waits of the compiler's only get stricter.
__device__ __forceinline__ void dma16(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :: "s"(lds), "v"(off), "s"(base) );
}
// the same with the lanes of `live`: all or none, so that a loop body needs no branch around its copies
// (called where every lane of the wave is active)
__device__ __forceinline__ void dma16_if(const char* base, uint32_t off, uint32_t lds, uint32_t live) {
  asm volatile("s_mov_b32 m0, %0\n\ts_mov_b32 exec_lo, %3\n\ts_mov_b32 exec_hi, %3\n\t"
               "global_load_lds_dwordx4 %1, %2\n\ts_mov_b64 exec, -1"
               :: "s"(lds), "v"(off), "s"(base), "s"(live) );
}
__device__ __forceinline__ void dma16_at(const char* addr, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(lds), "v"(addr) );
}
// Every copy of this wave has landed and its LDS reads are back; then all waves meet. Memory accesses
// stay on their side.
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
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

  // j-th load of a whole k tile
  __device__ __forceinline__ void one(int j, const char* base, const char* alt, uint32_t lds_wave, uint32_t live) const {
    dma16_if(is_alt(j) ? alt : base, off[j], lds_wave + j * NT * 16, live);
  }
  __device__ __forceinline__ void all(const char* base, const char* alt, uint32_t lds_wave) const {
#pragma unroll
    for (int j = 0; j < J; ++j) dma16(is_alt(j) ? alt : base, off[j], lds_wave + j * NT * 16);
  }
  // a k tile that ends inside: chunks from krem on come from the zeros
  __device__ __forceinline__ void tail(const char* base, const char* alt, uint32_t lds_wave, int t, int krem) const {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const char* g = (is_alt(j) ? alt : base) + off[j];
      dma16_at(kpos(j, t) < krem ? g : (const char*)zeros16, lds_wave + j * NT * 16);
    }
  }
};

// Fragments of a wave's rows [row0, row0 + 16 COUNT) of one side. Everything lane-dependent sits in a few
// base addresses (bytes of LDS, moved between the buffers by one add each); fragment, k half and
// row block are immediate offsets.
template <int LAYOUT, int R, int COUNT, bool DUAL>
struct Frags {
  static constexpr int NB = LAYOUT == KC ? 2 : COUNT;
  uint32_t at[NB];
  // first: LDS address of the image; w: this wave's position along the side, of `waves`
  __device__ __forceinline__ void init(uint32_t first, int w, int lane) {
    if constexpr (LAYOUT == KC) {
      const int row0 = DUAL ? row_dual(w, 0) : w * COUNT * 16;
      const uint32_t a0 = first + (uint32_t)(row0 + (lane & 15)) * 128u;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) at[kk] = a0 + 16u * (uint32_t)((kk * 4 + (lane >> 4)) ^ (lane & 7));
    } else {
      const int k = 8 * (lane >> 4) + ((lane & 15) >> 2);
#pragma unroll
      for (int i = 0; i < COUNT; ++i) {
        const int chunk = (((w * COUNT + i) * 2) ^ (2 * ks_h<R>(k))) + ((lane & 3) >> 1);
        at[i] = first + (uint32_t)(k * R + 8 * chunk + 4 * (lane & 1)) * 2u;
      }
    }
  }
  // DUAL: COUNT / 2 blocks of gate rows, then the up rows of the same columns
  __device__ __forceinline__ static int row_dual(int w, int i) {
    const int col = w * (COUNT / 2) * 16 + (i % (COUNT / 2)) * 16;
    return ((col >> 6) << 7) + (i >= COUNT / 2 ? 64 : 0) + (col & 63);
  }
  __device__ __forceinline__ bf16x8 get(int i, int kk) const {
    typedef __attribute__((address_space(3))) const bf16x8 LV;
    if constexpr (LAYOUT == KC) {
      // DUAL: a wave's columns lie in one block of 64, so its rows differ from row_dual(w, 0) by constants
      const uint32_t o = DUAL ? (uint32_t)((i % (COUNT / 2)) * 16 + (i >= COUNT / 2 ? 64 : 0)) * 128u : (uint32_t)i * 2048u;
      return *(LV*)(uintptr_t)(at[kk] + o);
    } else {
      typedef __attribute__((address_space(3))) short4_t TV;
      const uint32_t p = at[i] + (uint32_t)kk * (32u * R * 2u);
      const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TV*)(uintptr_t)p);
      const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TV*)(uintptr_t)(p + 8u * R));
      typedef short short8_t __attribute__((ext_vector_type(8)));
      const short8_t v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      return __builtin_bit_cast(bf16x8, v);
    }
  }
  __device__ __forceinline__ void move(uint32_t bytes) {
#pragma unroll
    for (int i = 0; i < NB; ++i) at[i] += bytes;
  }
};

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

// k tiles are double buffered. While tile t is multiplied, tile t + 1 is on its way or has landed;
// after the barrier in the middle of tile t nobody reads its buffer any more (the fragments of its
// second half are in registers), so the copies of tile t + 2 go out there, between the MFMAs, and the
// first fragments of tile t + 1 are read: one barrier a tile, a whole tile's time for the copies,
// and no MFMA waits on an LDS read that was not issued half a tile earlier.
template <int LM, int LN, int TM, int TN, int WM, int WN, bool DUAL, class Epi>
__global__ void __launch_bounds__(64 * WM * WN, TM * TN > 128 * 128 ? 1 : 2) gemm16_kernel(const Args a, const Epi epi) {
  constexpr int NT = 64 * WM * WN, WTM = TM / WM, WTN = TN / WN, MI = WTM / 16, NI = WTN / 16;
  constexpr int BUF = (TM + TN) * BK;  // elements of one buffer
  __shared__ __attribute__((aligned(128))) u16 lds[2 * BUF];
  int batch, split, mt, nt;
  tile_of(a, batch, split, mt, nt);
  batch = __builtin_amdgcn_readfirstlane(batch);  // (divisions leave uniform values in vector registers)
  split = __builtin_amdgcn_readfirstlane(split);
  mt = __builtin_amdgcn_readfirstlane(mt);
  nt = __builtin_amdgcn_readfirstlane(nt);
  const int M = __builtin_amdgcn_readfirstlane(a.dyn_m ? *a.dyn_m : a.M);
  const int K = __builtin_amdgcn_readfirstlane(a.dyn_k ? *a.dyn_k : a.K);
  const int x0m = mt * TM, x0n = nt * (DUAL ? TN / 2 : TN);
  if (x0m >= M) return;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wave % WM, wn = wave / WM;

  Stage<LM, TM, NT, false> sm;
  Stage<LN, TN, NT, DUAL> sn;
  sm.init(a.m, x0m, t);
  sn.init(a.n, x0n, t);
  const int64_t tm0 = a.m.bs * batch + (LM == KC ? (int64_t)x0m * a.m.ld : x0m);
  const int64_t tn0 = a.n.bs * batch + (LN == KC ? (int64_t)x0n * a.n.ld : x0n);
  const int64_t stepm = LM == KC ? BK : BK * a.m.ld, stepn = LN == KC ? BK : BK * a.n.ld;

  // k tiles in order: the segments' last, partial tiles first (at most two: they go out ahead of the
  // loop, which then copies whole tiles only), then the whole tiles of every segment
  const int full = K / BK, parts = K % BK ? a.nseg : 0, total = full * a.nseg + parts;
  const int per = (total + a.splits - 1) / a.splits;
  const int it0 = __builtin_amdgcn_readfirstlane(split * per);
  const int it1 = __builtin_amdgcn_readfirstlane(min(total, it0 + per));

  f32x4 acc[NI][MI];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const char *pm = nullptr, *pn = nullptr, *pa = nullptr;  // the next tile to copy
  int seg, kp;
  auto locate = [&](int it) {
    seg = __builtin_amdgcn_readfirstlane(it < parts ? it : full > 0 ? (it - parts) / full : 0);
    kp = it < parts ? full : it - parts - seg * full;
    const u16* bm = seg == 0 ? a.m.p[0] : seg == 1 ? a.m.p[1] : a.m.p[2];
    const u16* bn = seg == 0 ? a.n.p[0] : seg == 1 ? a.n.p[1] : a.n.p[2];
    pm = (const char*)(bm + tm0 + kp * stepm);
    pn = (const char*)(bn + tn0 + kp * stepn);
    if (DUAL) pa = (const char*)(a.n.alt + tn0 + kp * stepn);
  };
  const uint32_t ldsb = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) u16*)lds;
  const uint32_t lds0 = ldsb + (uint32_t)wave * 1024u;
  auto issue = [&](uint32_t l) {
    if (kp < full) {
      sm.all(pm, nullptr, l);
      sn.all(pn, pa, l + TM * BK * 2);
    } else {
      sm.tail(pm, nullptr, l, t, K - full * BK);
      sn.tail(pn, pa, l + TM * BK * 2, t, K - full * BK);
    }
  };
  Frags<LM, TM, MI, false> gm;
  Frags<LN, TN, NI, DUAL> gn;
  gm.init(ldsb, wm, lane);
  gn.init(ldsb + TM * BK * 2, wn, lane);

  if (it0 < it1) {
    constexpr int NF = MI + NI, NQ = sm.J + sn.J, NX = NI * MI;
    bf16x8 fm[2][MI], fn[2][NI];
    locate(it0);
    issue(lds0);
    if (it0 + 1 < it1) {
      locate(it0 + 1);
      tile_barrier();
      issue(lds0 + BUF * 2);
    } else {
      tile_barrier();
    }
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      if (f < MI) fm[0][f < MI ? f : 0] = gm.get(f, 0);
      else fn[0][f < MI ? 0 : f - MI] = gn.get(f - MI, 0);
    }
    locate(it0 + 2);
    uint32_t lq = lds0, hop = BUF * 2;  // where the next copies go; to the other buffer
    for (int it = it0; it < it1; ++it) {
      const uint32_t live = (uint32_t)__builtin_amdgcn_readfirstlane(it + 2 < it1 ? -1 : 0);
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        if (f < MI) fm[1][f < MI ? f : 0] = gm.get(f, 1);
        else fn[1][f < MI ? 0 : f - MI] = gn.get(f - MI, 1);
#pragma unroll
        for (int x = f * NX / NF; x < (f + 1) * NX / NF; ++x)
          acc[x / MI][x % MI] = mfma16(fn[0][x / MI], fm[0][x % MI], acc[x / MI][x % MI]);
      }
      tile_barrier();
      gm.move(hop);
      gn.move(hop);
#pragma unroll
      for (int f = 0; f < NF; ++f) {
#pragma unroll
        for (int q = f * NQ / NF; q < (f + 1) * NQ / NF; ++q) {
          if (q < sm.J) sm.one(q < sm.J ? q : 0, pm, nullptr, lq, live);
          else sn.one(q < sm.J ? 0 : q - sm.J, pn, pa, lq + TM * BK * 2, live);
        }
        // (of the last tile: not used)
        if (f < MI) fm[0][f < MI ? f : 0] = gm.get(f, 0);
        else fn[0][f < MI ? 0 : f - MI] = gn.get(f - MI, 0);
#pragma unroll
        for (int x = f * NX / NF; x < (f + 1) * NX / NF; ++x)
          acc[x / MI][x % MI] = mfma16(fn[1][x / MI], fm[1][x % MI], acc[x / MI][x % MI]);
      }
      lq += hop;
      hop = 0u - hop;
      if (++kp == full) {
        locate(it + 3);
      } else {
        pm += stepm * 2;
        pn += stepn * 2;
        if (DUAL) pa += stepn * 2;
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

// Output tiles. Both shapes run four waves, two along each side.
enum { T128 = 128, T256 = 256 };

template <int LM, int LN, int TM, int TN, int WM, int WN, bool DUAL = false, class Epi>
void launch_tile(Args a, const Epi& e, hipStream_t stream) {
  a.tiles_m = cdiv(a.M, TM);
  a.tiles_n = cdiv(a.N, DUAL ? TN / 2 : TN);
  const int64_t tiles = a.sym ? (int64_t)a.tiles_m * (a.tiles_m + 1) / 2 : (int64_t)a.tiles_m * a.tiles_n;
  const int64_t blocks = tiles * a.splits * a.batch;
  if (blocks <= 0) return;
  gemm16_kernel<LM, LN, TM, TN, WM, WN, DUAL, Epi><<<dim3((unsigned)blocks), dim3(64 * WM * WN), 0, stream>>>(a, e);
}

template <int LM, int LN, bool DUAL = false, class Epi>
void launch(int tile, const Args& a, const Epi& e, hipStream_t stream) {
  if (tile == T256) launch_tile<LM, LN, 256, 256, 2, 2, DUAL>(a, e, stream);
  else launch_tile<LM, LN, 128, 128, 2, 2, DUAL>(a, e, stream);
}

// How to run a product: the tile and the k splits with the least estimated time. One 64-wide k tile
// costs a block about 1.5 us at 256x256 (one block a CU) and 0.9 us at 128x128 (two a CU); a block's
// start and its epilogue cost about three of them; splits pay for their slabs' way through memory.
struct Plan {
  int tile, splits;
};
inline Plan plan(int64_t M, int64_t N, int64_t K, int nseg, int batch, bool sym, bool may_split) {
  Plan best{T128, 1};
  double best_t = 1e30;
  const int64_t kt = (int64_t)cdiv(K, BK) * nseg;
  const int cus = device_cu_count();
  for (int tile : {T256, T128}) {
    const int64_t tm = cdiv(M, tile), tn = cdiv(N, tile);
    const int64_t tiles = (sym ? tm * (tm + 1) / 2 : tm * tn) * batch;
    const int64_t slots = tile == T256 ? cus : 2 * cus;
    const double unit = tile == T256 ? 1.5 : 0.9;
    for (int s = 1; s <= 64 && (s == 1 || (may_split && kt / s >= 4)); ++s) {
      const int64_t rounds = (tiles * s + slots - 1) / slots;
      double t = (double)rounds * ((double)((kt + s - 1) / s) + 3.0) * unit;
      if (s > 1) t += 3.0 + (double)M * N * batch * (s + 0.5) * 8.0 / 4e6;
      if (t < best_t) {
        best_t = t;
        best = {tile, s};
      }
    }
  }
  return best;
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

// A product rounded once into 16-bit outputs (one or two batch entries), split along k when its
// tiles alone leave CUs idle.
template <int LM, int LN>
void product(Args a, u16* out0, u16* out1, int64_t ldo, float alpha, const float* dev_alpha, c10::Device dev,
             hipStream_t stream) {
  const Plan p = plan(a.M, a.N, a.K, a.nseg, a.batch, false, true);
  a.splits = p.splits;
  if (p.splits == 1) {
    launch<LM, LN>(p.tile, a, EpiStore{{out0, out1}, ldo, alpha, dev_alpha}, stream);
    return;
  }
  const int64_t ld = up8(a.N), stride = (int64_t)a.M * ld;
  at::Tensor slab = at::empty({a.batch * a.splits * stride}, at::TensorOptions().device(dev).dtype(at::kFloat));
  launch<LM, LN>(p.tile, a, EpiSlab{slab.data_ptr<float>(), ld, stride, a.splits, 0}, stream);
  slab_sum<<<dim3(cdiv((int64_t)a.M * ((a.N + 3) / 4), 256), a.batch), 256, 0, stream>>>(
      slab.data_ptr<float>(), a.splits, stride, ld, a.M, a.N, out0, out1, ldo, alpha, dev_alpha);
}

}  // namespace g16
MIHVD_OPNS_END
