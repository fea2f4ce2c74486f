// Matrix-product core of the transformer-step operators (linear_ce.hip, gated_ffn.hip,
// newton_schulz.hip): 16-bit operands (bf16, or fp16 in a -DMIHVD_F16 build), fp32 accumulation,
// with the operator's own work in the epilogue.
//
//   out[m][n] = sum over segments s and k < K of  Pm_s(m, k) * Pn_s(n, k)
//
// Each side is stored K-contiguous ("KC", [row][k]) or K-strided ("KS", [k][row]), so no operand is
// ever transposed in memory: forward products are KC x KC, products with a weight along its other
// axis KC x KS, weight gradients KS x KS. Segments concatenate products along k (the two halves of
// a gated input gradient).
//
// The n side feeds the MFMA's A operand and the m side its B operand, so a lane's four accumulators
// are four consecutive n of one m (v_mfma_f32_16x16x32: C[4*(l>>4)+i][l&15]): packed 8-byte stores
// along the output rows, and a reduction over n stays in the lane but for two exchanges.
//
// Staging is global_load_lds_dwordx4 into swizzled LDS images (two buffers; four at 64x64). Out-of-range rows
// are clamped to the last row (their products only reach outputs that are never stored); k positions
// past K are read from a page of zeros on both sides.
//
// What a caller guarantees (transformer_ops.cpp packs what does not fit): 16-byte aligned bases, leading
// dimensions and KS extents that are multiples of 8 elements, KC rows that hold zeros (or any
// finite values against zeros) from K to the next multiple of 8.
//
// Bound by the matrix pipe and by what a tile's end costs: plain bf16 products of 8192 x 8192 at 256x256 run at
// 0.97, 1.20 and 1.45 PFLOP/s for K = 768, 2048 and 8192 (the card's library: 1.10, 1.40 and 1.40). A wave's
// 128x128 part reads 32 KB of LDS for 128 MFMAs, which is half the LDS's rate; at 64x64 a wave the LDS
// reads and the copies into it together take as long as the MFMAs, hence 256x256 wherever there are tiles
// enough. Giving every block an equal run of k tiles across output tiles was slower at every shape tried
// (2048 x 5632 x 16384: 427 us against 357): blocks at different k share nothing in L2.
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
  const u16* p[2] = {nullptr, nullptr};           // one base per segment, or plane
  const u16* alt = nullptr;                       // DUAL: the second matrix of interleaved rows
  int64_t ld = 0;                                 // elements between rows (KC) / between k (KS)
  int64_t bs = 0;                                 // elements between batch entries
  int ext = 0;                                    // rows (KC); storage extent, a multiple of 8 (KS)
};

// A ragged batch (template parameter RAG): entry b is a matrix of `rows` x len[b], in planes of that size
// one behind the other from element off[b] on.
//   RAG 1: both sides are such matrices along k (K = len[b]);  RAG 2: the n side is one, K-strided (N = len[b])
constexpr int RAG_MAX = 32;
struct Ragged {
  int rows = 0, count = 0;
  int len[RAG_MAX];
  int64_t off[RAG_MAX];
  int start[RAG_MAX + 1];  // RAG 2: first tile of each entry; filled by launch()
};

// k splits of a product whose rows are counted on the device, by the count: the split with the least
// estimated time (the terms of plan(), in 0.01 us) of those whose slabs fit.
struct SplitRule {
  int cap = 0;            // row tiles times splits that the slabs hold
  int tile, tn, kt, cus;  // output tile, tiles along the columns, k tiles, compute units
  int unit1, unit2, end;  // a k tile with one and with two blocks on a CU (0: never two), a tile's end
  int N;
  int* chosen;            // where the kernel leaves its choice for the one that sums the slabs
};
// Every lane of a wave prices one split; all waves get the same answer.
__device__ __forceinline__ int pick_splits(const SplitRule& r, int M) {
  const int lane = threadIdx.x & 63, s = lane + 1;
  const int64_t tm = (M + r.tile - 1) / r.tile, tiles = tm * r.tn * s;
  const bool two = r.unit2 && tiles > r.cus;
  const int slots = two ? 2 * r.cus : r.cus;
  const int64_t rounds = (tiles + slots - 1) / slots;
  int64_t cost = rounds * ((int64_t)((r.kt + s - 1) / s) * (two ? r.unit2 : r.unit1) + r.end);
  cost += (int64_t)M * r.N * (2 * s + 1) / 10000;  // 8 (s + 1/2) bytes a value at 4 TB/s
  if (s > 1 && (r.kt / s < 4 || tm * s > r.cap)) cost = INT64_MAX >> 8;
  int64_t key = cost * 64 + lane;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = __shfl_xor(key, d);
    key = o < key ? o : key;
  }
  return __builtin_amdgcn_readfirstlane((int)(key & 63)) + 1;
}

struct Args {
  Side m, n;
  int M = 0, N = 0, K = 0;  // K: per segment
  int nseg = 1, batch = 1, splits = 1;
  int sym = 0;                  // out is symmetric (M == N): only tiles with nt >= mt run
  const int* dyn_m = nullptr;   // device count that replaces M (tiles past it do not run)
  const int* dyn_k = nullptr;   // device count that replaces K
  SplitRule rule;               // with dyn_m: how the kernel itself chooses the k splits (rule.cap 0: `splits`)
  int tiles_m = 0, tiles_n = 0; // filled by launch()
};

// What an epilogue sees of its wave: the wave's first m and n, and the tile it belongs to.
struct Ctx {
  int m0, n0;      // origin of the wave tile (DUAL: n0 in columns of one matrix)
  int M, N;        // bounds (M after dyn_m)
  int mt, nt;      // tile indices
  int wm, wn;      // wave position in the tile
  int batch, split, lane;
  int64_t off;     // RAG 2: the entry's first element and row length
  int len;
  u16* stage;      // this wave's LDS for RowStage
};

// 16 rows of 16-bit results on their way out, in LDS that only this wave uses: a lane's four
// consecutive values go in where the accumulators hold them (16 rows, 32 bytes of each), and come back
// as 16 bytes of a row, so that a store instruction writes whole rows of the wave's tile. Rows are
// padded by 16 bytes: both directions are free of bank conflicts.
template <int COLS>
struct RowStage {
  static constexpr int RS = COLS + 8, CH = COLS / 8, GETS = 16 * CH / 64;
  u16* p;
  int lane;
  __device__ __forceinline__ void put(int i, uint2 v) const {
    *reinterpret_cast<uint2*>(p + (lane & 15) * RS + i * 16 + 4 * (lane >> 4)) = v;
  }
  __device__ __forceinline__ uint2 take(int i) const {
    return *reinterpret_cast<const uint2*>(p + (lane & 15) * RS + i * 16 + 4 * (lane >> 4));
  }
  __device__ __forceinline__ void set(int g, uint4 v) const { *reinterpret_cast<uint4*>(p + row(g) * RS + col()) = v; }
  __device__ __forceinline__ static void turn() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
  __device__ __forceinline__ int row(int g) const { return lane / CH + g * (64 / CH); }
  __device__ __forceinline__ int col() const { return (lane % CH) * 8; }
  __device__ __forceinline__ uint4 get(int g) const {
    return *reinterpret_cast<const uint4*>(p + row(g) * RS + col());
  }
};

// Row permutation of a KS image: 16-byte chunks of k row `k` are XORed with 2*h(k), so that the
// eight k rows a half wave reads with ds_read_b64_tr_b16 land in different 32-byte bank groups.
template <int R>
__device__ __forceinline__ int ks_h(int k) {
  if constexpr (R >= 128) return (k & 3) | (((k >> 3) & 1) << 2);
  else return ((k >> 1) & 1) | (((k >> 3) & 1) << 1);
}

// A wave-uniform value into a scalar register. In asm because the compiler drops its own readfirstlane
// where it knows the value to be uniform, and may then keep it, and what follows from it, in vector
// registers. The waits: one state between a vector instruction that writes x and the lane read (gfx940
// and later need it), five before a memory access that takes the result as its base.
__device__ __forceinline__ int uni(int x) {
  int r;
  asm("s_nop 1\n\tv_readfirstlane_b32 %0, %1\n\ts_nop 4" : "=s"(r) : "v"(x));
  return r;
}

// Direct global -> LDS copies of 16 bytes a lane (lane l's land at lds + 16 l; lds is wave-uniform).
// Written in asm because the compiler, which cannot tell the two LDS buffers apart, waits for every
// copy in flight before any LDS read; the kernel's own s_waitcnt before the barrier is the wait these
// need. They have no destination registers, and later waits of the compiler's only get stricter.
__device__ __forceinline__ void dma16(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2"
               :: "s"(lds), "v"(off), "s"(base) );
}
__device__ __forceinline__ void dma16_if(const char* base, uint32_t off, uint32_t lds, uint64_t live) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\ts_mov_b64 exec, %3\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b64 exec, -1"
               :: "s"(lds), "v"(off), "s"(base), "s"(live));
}
__device__ __forceinline__ void dma16_at(const char* addr, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(lds), "v"(addr) );
}
// f(0), f(1), ... f(N - 1) with constants, whatever the unroller thinks of the size
template <int N, class F, int I = 0>
__device__ __forceinline__ void unroll(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    unroll<N, F, I + 1>(static_cast<F&&>(f));
  }
}

// Four MFMAs that accumulate in place. In asm so that the accumulators stay where they are (the compiler
// moves them between registers when they fill the accumulation file) and the order of MFMAs, copies
// and LDS reads stays as written; s_nop 1 covers operands that a vector instruction wrote just before.
// BIG: 256 accumulators, in the accumulation registers; else any vector registers.
#ifdef MIHVD_F16
#define MIHVD_G16_MFMA "v_mfma_f32_16x16x32_f16"
#else
#define MIHVD_G16_MFMA "v_mfma_f32_16x16x32_bf16"
#endif
template <bool BIG>
__device__ __forceinline__ void mfma4(f32x4& c0, f32x4& c1, f32x4& c2, f32x4& c3, const bf16x8& a, const bf16x8& b0,
                                      const bf16x8& b1, const bf16x8& b2, const bf16x8& b3) {
#define MIHVD_G16_ASM                                                                                           \
  "s_nop 1\n\t" MIHVD_G16_MFMA " %0, %4, %5, %0\n\t" MIHVD_G16_MFMA " %1, %4, %6, %1\n\t" MIHVD_G16_MFMA       \
  " %2, %4, %7, %2\n\t" MIHVD_G16_MFMA " %3, %4, %8, %3"
  if constexpr (BIG)
    asm volatile(MIHVD_G16_ASM : "+a"(c0), "+a"(c1), "+a"(c2), "+a"(c3) : "v"(a), "v"(b0), "v"(b1), "v"(b2), "v"(b3));
  else
    asm volatile(MIHVD_G16_ASM : "+v"(c0), "+v"(c1), "+v"(c2), "+v"(c3) : "v"(a), "v"(b0), "v"(b1), "v"(b2), "v"(b3));
#undef MIHVD_G16_ASM
}
// Two by two, for waves of 32 x 32.
__device__ __forceinline__ void mfma2x2(f32x4& c00, f32x4& c01, f32x4& c10, f32x4& c11, const bf16x8& a0, const bf16x8& a1,
                                        const bf16x8& b0, const bf16x8& b1) {
  asm volatile("s_nop 1\n\t" MIHVD_G16_MFMA " %0, %4, %6, %0\n\t" MIHVD_G16_MFMA " %1, %4, %7, %1\n\t" MIHVD_G16_MFMA
               " %2, %5, %6, %2\n\t" MIHVD_G16_MFMA " %3, %5, %7, %3"
               : "+v"(c00), "+v"(c01), "+v"(c10), "+v"(c11) : "v"(a0), "v"(a1), "v"(b0), "v"(b1));
}
// The same with one or two of the tile's copies between them, each no longer than an MFMA: from base +
// off to LDS l + at, by all lanes or none (`live`: a loop body then needs no branch around its copies;
// every lane of the wave is active here).
#define MIHVD_G16_COPY(OFF, BASE)                                                                       \
  "s_mov_b64 exec, %10\n\tglobal_load_lds_dwordx4 " OFF ", " BASE "\n\ts_mov_b64 exec, -1\n\t"
template <bool BIG>
__device__ __forceinline__ void mfma4_copy(f32x4& c0, f32x4& c1, f32x4& c2, f32x4& c3, const bf16x8& a, const bf16x8& b0,
                                           const bf16x8& b1, const bf16x8& b2, const bf16x8& b3, uint32_t l, uint64_t live,
                                           int at, uint32_t off, const char* base) {
#define MIHVD_G16_ASM                                                                                              \
  "s_nop 1\n\t" MIHVD_G16_MFMA " %0, %4, %5, %0\n\ts_add_u32 m0, %9, %11\n\t" MIHVD_G16_MFMA                     \
  " %1, %4, %6, %1\n\t" MIHVD_G16_COPY("%12", "%13") MIHVD_G16_MFMA " %2, %4, %7, %2\n\t" MIHVD_G16_MFMA     \
  " %3, %4, %8, %3"
  if constexpr (BIG)
    asm volatile(MIHVD_G16_ASM : "+a"(c0), "+a"(c1), "+a"(c2), "+a"(c3)
                 : "v"(a), "v"(b0), "v"(b1), "v"(b2), "v"(b3), "s"(l), "s"(live), "n"(at), "v"(off), "s"(base) : "scc");
  else
    asm volatile(MIHVD_G16_ASM : "+v"(c0), "+v"(c1), "+v"(c2), "+v"(c3)
                 : "v"(a), "v"(b0), "v"(b1), "v"(b2), "v"(b3), "s"(l), "s"(live), "n"(at), "v"(off), "s"(base) : "scc");
#undef MIHVD_G16_ASM
}
template <bool BIG>
__device__ __forceinline__ void mfma4_copy2(f32x4& c0, f32x4& c1, f32x4& c2, f32x4& c3, const bf16x8& a, const bf16x8& b0,
                                            const bf16x8& b1, const bf16x8& b2, const bf16x8& b3, uint32_t l,
                                            uint64_t live, int at, uint32_t off, const char* base, int at2, uint32_t off2,
                                            const char* base2) {
#define MIHVD_G16_ASM                                                                                              \
  "s_nop 1\n\t" MIHVD_G16_MFMA " %0, %4, %5, %0\n\ts_add_u32 m0, %9, %11\n\t" MIHVD_G16_MFMA                     \
  " %1, %4, %6, %1\n\t" MIHVD_G16_COPY("%12", "%13") MIHVD_G16_MFMA                                         \
  " %2, %4, %7, %2\n\ts_add_u32 m0, %9, %14\n\t" MIHVD_G16_COPY("%15", "%16") MIHVD_G16_MFMA " %3, %4, %8, %3"
  if constexpr (BIG)
    asm volatile(MIHVD_G16_ASM : "+a"(c0), "+a"(c1), "+a"(c2), "+a"(c3)
                 : "v"(a), "v"(b0), "v"(b1), "v"(b2), "v"(b3), "s"(l), "s"(live), "n"(at), "v"(off), "s"(base), "n"(at2),
                   "v"(off2), "s"(base2) : "scc");
  else
    asm volatile(MIHVD_G16_ASM : "+v"(c0), "+v"(c1), "+v"(c2), "+v"(c3)
                 : "v"(a), "v"(b0), "v"(b1), "v"(b2), "v"(b3), "s"(l), "s"(live), "n"(at), "v"(off), "s"(base), "n"(at2),
                   "v"(off2), "s"(base2) : "scc");
#undef MIHVD_G16_ASM
}
// The matrix pipe's results may be read after this (16 wait states; the longest needed is 11).
template <bool BIG>
__device__ __forceinline__ void mfma_done(f32x4& c0, f32x4& c1, f32x4& c2, f32x4& c3) {
  if constexpr (BIG) asm volatile("s_nop 15" : "+a"(c0), "+a"(c1), "+a"(c2), "+a"(c3));
  else asm volatile("s_nop 15" : "+v"(c0), "+v"(c1), "+v"(c2), "+v"(c3));
}
// Keeps the accumulators of row block j where they are until an epilogue comes to them (left alone, the
// compiler copies all of them to vector registers at once, which do not suffice).
template <int NI, int MI>
__device__ __forceinline__ void pin(f32x4 (&acc)[NI][MI], int j) {
  if constexpr (NI == 2) {
    asm volatile("" : "+v"(acc[0][j]), "+v"(acc[1][j]));
    return;
  }
#pragma unroll
  for (int i = 0; i + 3 < NI; i += 4) {
    if constexpr (NI * MI > 16) asm volatile("" : "+a"(acc[i][j]), "+a"(acc[i + 1][j]), "+a"(acc[i + 2][j]), "+a"(acc[i + 3][j]));
    else asm volatile("" : "+v"(acc[i][j]), "+v"(acc[i + 1][j]), "+v"(acc[i + 2][j]), "+v"(acc[i + 3][j]));
  }
}
// Every copy of this wave has landed and its LDS reads are back; then all waves meet. Memory accesses
// stay on their side.
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The same with the newest N copies (of later tiles) still on their way.
template <int N>
__device__ __forceinline__ void tile_barrier_but() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(N) : "memory");
}
__device__ __forceinline__ void tile_barrier_landed() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
__device__ __forceinline__ void copies_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// One side's staging of an [R x 64] (KC) or [64 x R] (KS) tile by NT threads.
template <int LAYOUT, int R, int NT, bool DUAL>
struct Stage {
  static constexpr int J = R * 8 / NT;
  static_assert(J * NT == R * 8 && NT % 64 == 0, "whole chunks per thread");
  uint32_t off[J];

  __device__ __forceinline__ void init(int64_t ld, int ext, int x0, int t) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int i = t + j * NT;
      if constexpr (LAYOUT == KC) {
        const int row = i >> 3, src = (i & 7) ^ (row & 7);
        const int r = DUAL ? ((row >> 7) << 6) + (row & 63) : row;  // 64 rows of p, 64 of alt, ...
        off[j] = (uint32_t)min(r, ext - 1 - x0) * (uint32_t)ld * 2u + (uint32_t)src * 16u;
      } else {
        constexpr int RC = R / 8;
        const int k = i / RC, src = (i % RC) ^ (2 * ks_h<R>(k));
        off[j] = (uint32_t)k * (uint32_t)ld * 2u + (uint32_t)min(8 * src, ext - 8 - x0) * 2u;
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
  // pl: the image `pl` rows-images further on (PL 2: the low halves)
  __device__ __forceinline__ bf16x8 get(int i, int kk, int pl = 0) const {
    typedef __attribute__((address_space(3))) const bf16x8 LV;
    if constexpr (LAYOUT == KC) {
      // DUAL: a wave's columns lie in one block of 64, so its rows differ from row_dual(w, 0) by constants
      const uint32_t o = DUAL ? (uint32_t)((i % (COUNT / 2)) * 16 + (i >= COUNT / 2 ? 64 : 0)) * 128u : (uint32_t)i * 2048u;
      return *(LV*)(uintptr_t)(at[kk] + o + (uint32_t)pl * (R * 128u));
    } else {
      typedef __attribute__((address_space(3))) short4_t TV;
      const uint32_t p = at[i] + (uint32_t)kk * (32u * R * 2u) + (uint32_t)pl * (R * 128u);
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

// One output tile of one k split: where it is and its k tiles [it, end).
struct Tile {
  int batch, split, mt, nt, it, end;
  int K, N;  // of the batch entry
};

// Tile order. Blocks are persistent: the blocks of one XCD (every eighth block) walk a contiguous
// run of tiles together, in groups of eight m tiles, so that the tiles an XCD has in flight share rows
// of both operands in its L2. `l` counts within the XCD's run; false past its end.
template <int RAG, int TN>
__device__ __forceinline__ bool tile_at(const Args& a, const Ragged& g, int tiles_m, int splits, int K, int l, Tile& t) {
  const int tiles = a.sym ? tiles_m * (tiles_m + 1) / 2 : tiles_m * a.tiles_n;
  const int nb = RAG == 2 ? g.start[g.count] : tiles * splits * a.batch, x = blockIdx.x & 7;
  const int q = nb >> 3, r = nb & 7;
  if (l >= q + (x < r ? 1 : 0)) return false;
  // (an XCD's run goes up through the entries: the search starts where the last one ended)
  int pos = x * q + min(x, r) + l, mt, nt, batch = RAG == 2 ? t.batch : 0, split = 0, tiles_n = a.tiles_n;
  t.K = K;
  t.N = a.N;
  if constexpr (RAG == 2) {
    while (pos >= g.start[batch + 1]) ++batch;
    pos -= g.start[batch];
    t.N = g.len[batch];
    tiles_n = (t.N + TN - 1) / TN;
  } else if (a.batch > 1 || splits > 1) {
    const int e = pos / tiles;
    pos -= e * tiles;
    batch = e / splits;
    split = e - batch * splits;
    if constexpr (RAG == 1) t.K = g.len[batch];
  } else if constexpr (RAG == 1) {
    t.K = g.len[0];
  }
  if (a.sym) {
    mt = 0;
    while (pos >= tiles_m - mt) {
      pos -= tiles_m - mt;
      ++mt;
    }
    nt = mt + pos;
  } else {
    constexpr int G = 8;
    const int grp = pos / (G * tiles_n), first = grp * G;
    const int gs = min(G, tiles_m - first);
    pos -= grp * G * tiles_n;
    nt = pos / gs;
    mt = first + pos - nt * gs;
  }
  t.batch = uni(batch);
  t.split = uni(split);
  t.mt = uni(mt);
  t.nt = uni(nt);
  t.K = uni(t.K);
  const int kts = (t.K + BK - 1) / BK * a.nseg;
  t.it = splits == 1 ? 0 : uni((int)((int64_t)kts * t.split / splits));
  t.end = splits == 1 ? kts : uni((int)((int64_t)kts * (t.split + 1) / splits));
  return true;
}

// k tiles go through S buffers. While tile t is multiplied, the tiles up to t + S - 1 are on their way or
// have landed; after the barrier in the middle of tile t nobody reads its buffer any more (the
// fragments of its second half are in registers), so the copies of tile t + S go out there, between the
// MFMAs, and the first fragments of tile t + 1 are read: one barrier a tile, S - 1 tiles' time for the
// copies, and no MFMA waits on an LDS read that was not issued half a tile earlier.
//
// The stream of k tiles runs on from one output tile to the next: while the epilogue works, the next
// output tile's first two k tiles are already in LDS and its first fragments in registers, and the
// epilogue's stores drain under the next products.
//
// PL 2: both sides are split values, in two planes (segments 0 and 1 of a side are its high and low
// halves), and the three products hi hi + hi lo + lo hi run on one staging of the four images: a third
// of the k tiles that three segments would take, two thirds of their LDS reads.
template <int LM, int LN, int TM, int TN, int S, int PL, bool DUAL, int RAG, class Epi>
__global__ void __launch_bounds__(256, TM * TN > 128 * 128 || PL == 2 ? 1 : 2)
    gemm16_kernel(const Args a, const typename std::conditional<RAG != 0, Ragged, int>::type rag, const Epi epi) {
  constexpr int WM = 2, WN = 2, NT = 64 * WM * WN, WTM = TM / WM, WTN = TN / WN, MI = WTM / 16, NI = WTN / 16;
  constexpr int BUF = PL * (TM + TN) * BK;  // elements of one buffer
  constexpr bool BIG = TM * TN > 128 * 128;
  constexpr int STAGE = 16 * (WTN + 8);  // a wave's RowStage
  __shared__ __attribute__((aligned(128))) u16 lds[S * BUF + WM * WN * STAGE];
  const int M = uni(a.dyn_m ? *a.dyn_m : a.M);
  const int K = uni(a.dyn_k ? *a.dyn_k : a.K);
  const int tiles_m = a.dyn_m ? (M + TM - 1) / TM : a.tiles_m;
  int splits = a.splits;
  if (a.rule.cap) {
    splits = pick_splits(a.rule, M);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.rule.chosen = splits;
  }
  const Ragged* gp = nullptr;
  if constexpr (RAG != 0) gp = &rag;
  const Ragged& g = *gp;  // (not read without RAG)
  const int hops = (int)(gridDim.x >> 3) + ((blockIdx.x & 7) < (gridDim.x & 7) ? 1 : 0);
  int l_mul = blockIdx.x >> 3, l_cpy = l_mul;  // the tile being multiplied, the tile being copied
  Tile cur, nxt;
  cur.batch = 0;
  if (!tile_at<RAG, TN>(a, g, tiles_m, splits, K, l_mul, cur)) return;
  const int t = threadIdx.x, lane = t & 63, wave = uni(t >> 6);
  const int wm = wave % WM, wn = wave / WM;

  Stage<LM, TM, NT, false> sm;
  Stage<LN, TN, NT, DUAL> sn;
  int64_t stepm = LM == KC ? BK : BK * a.m.ld, stepn = LN == KC ? BK : BK * a.n.ld;

  // The next k tile to copy: `run` whole ones lie ahead at (pm, pn), one step apart; then, with run == 0,
  // what `next_run` finds: a partial tile (krem > 0 of its k positions, none for a split without any k),
  // the next segment, the next output tile, or the end.
  const char *pm = nullptr, *pn = nullptr, *pa = nullptr, *pm2 = nullptr, *pn2 = nullptr;
  int run = 0, seg = 0, krem = 0;
  bool partial = false, more = true;
  auto locate = [&](int kp) {
    const int x0m = nxt.mt * TM, x0n = nxt.nt * (DUAL ? TN / 2 : TN);
    const int64_t len = RAG ? g.len[nxt.batch] : 0, plane = RAG ? len * g.rows : 0;
    const int64_t ldm = RAG == 1 ? len : a.m.ld, ldn = RAG ? len : a.n.ld;
    const int64_t tm0 = (RAG == 1 ? g.off[nxt.batch] : a.m.bs * nxt.batch) + (LM == KC ? (int64_t)x0m * ldm : x0m);
    const int64_t tn0 = (RAG ? g.off[nxt.batch] : a.n.bs * nxt.batch) + (LN == KC ? (int64_t)x0n * ldn : x0n);
    const u16* bm = seg == 0 ? a.m.p[0] : a.m.p[1];
    const u16* bn = seg == 0 ? a.n.p[0] : a.n.p[1];
    if constexpr (RAG == 2) stepn = LN == KC ? BK : BK * len;
    pm = (const char*)(bm + tm0 + kp * stepm);
    pn = (const char*)(bn + tn0 + kp * stepn);
    if (DUAL) pa = (const char*)(a.n.alt + tn0 + kp * stepn);
    if constexpr (PL == 2) {
      pm2 = RAG == 1 ? pm + plane * 2 : (const char*)(a.m.p[1] + tm0 + kp * stepm);
      pn2 = RAG ? pn + plane * 2 : (const char*)(a.n.p[1] + tn0 + kp * stepn);
    }
    const int whole = nxt.K / BK - kp;  // whole tiles of this segment from here on
    run = min(whole, nxt.end - nxt.it);
    partial = run == 0;
    krem = nxt.it < nxt.end ? nxt.K - kp * BK : 0;
    nxt.it += max(run, 1);
  };
  auto enter = [&]() {  // the copies reach output tile nxt
    const int len = RAG ? g.len[nxt.batch] : 0;
    sm.init(RAG == 1 ? len : a.m.ld, a.m.ext, nxt.mt * TM, t);
    sn.init(RAG ? len : a.n.ld, RAG == 2 ? len : a.n.ext, nxt.nt * (DUAL ? TN / 2 : TN), t);
    const int kt = (nxt.K + BK - 1) / BK;
    seg = a.nseg == 1 ? 0 : uni(kt > 0 ? nxt.it / kt : 0);
    locate(nxt.it - seg * kt);
  };
  auto next_run = [&]() {
    if (!more) return;
    if (nxt.it < nxt.end) {
      const int kt = (nxt.K + BK - 1) / BK, kp = nxt.it - seg * kt;
      if (kp == kt) ++seg;
      locate(kp == kt ? 0 : kp);
    } else {
      l_cpy += hops;
      more = tile_at<RAG, TN>(a, g, tiles_m, splits, K, l_cpy, nxt);
      if (more) enter();
    }
  };
  const uint32_t ldsb = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) u16*)lds;
  const uint32_t lds0 = ldsb + (uint32_t)wave * 1024u;
  auto step_on = [&](int64_t mask) {
    pm += (stepm * 2) & mask;
    pn += (stepn * 2) & mask;
    if (DUAL) pa += (stepn * 2) & mask;
    if (PL == 2) {
      pm2 += (stepm * 2) & mask;
      pn2 += (stepn * 2) & mask;
    }
  };
  constexpr uint32_t IMG_M = TM * BK * 2, IMG_N = TN * BK * 2;  // bytes of an image
  // the next k tile as a whole, ahead of the loop or where the run ends
  auto issue = [&](uint32_t l) -> bool {
    if (run == 0 && !partial) next_run();
    if (run > 0) {
      sm.all(pm, nullptr, l);
      if (PL == 2) sm.all(pm2, nullptr, l + IMG_M);
      sn.all(pn, pa, l + PL * IMG_M);
      if (PL == 2) sn.all(pn2, nullptr, l + PL * IMG_M + IMG_N);
      step_on(-1);
      --run;
      return true;
    }
    if (partial) {
      sm.tail(pm, nullptr, l, t, krem);
      if (PL == 2) sm.tail(pm2, nullptr, l + IMG_M, t, krem);
      sn.tail(pn, pa, l + PL * IMG_M, t, krem);
      if (PL == 2) sn.tail(pn2, nullptr, l + PL * IMG_M + IMG_N, t, krem);
      partial = false;
      return true;
    }
    return false;
  };
  Frags<LM, TM, MI, false> gm;
  Frags<LN, TN, NI, DUAL> gn;
  gm.init(ldsb, wm, lane);
  gn.init(ldsb + PL * IMG_M, wn, lane);

  f32x4 acc[NI][MI];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < MI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  clear();

  // A half tile: B4 blocks of four MFMAs (block b: accumulators from 4 (b / PR) on, product b % PR), among
  // which go the next half's NF fragment reads, all within the first three quarters so that none is
  // waited for at the barrier, and (second half) the NQ copies.
  constexpr int JM = decltype(sm)::J, JN = decltype(sn)::J, NF = PL * (MI + NI), NQ = PL * (JM + JN), NX = NI * MI;
  constexpr int PR = PL == 2 ? 3 : 1, B4 = NX / 4 * PR;
  auto ahead = [](int b) constexpr { return b * NF * 4 / (3 * B4) < NF ? b * NF * 4 / (3 * B4) : NF; };
  bf16x8 fm[2][PL][MI], fn[2][PL][NI];
  auto read = [&](int f, int set, int kk) {
    const int pl = f / (MI + NI), r = f % (MI + NI);
    if (r < MI) fm[set][pl][r < MI ? r : 0] = gm.get(r, kk, pl);
    else fn[set][pl][r < MI ? 0 : r - MI] = gn.get(r - MI, kk, pl);
  };
  // the copies of the last S - 2 tiles may be on their way across a barrier; not once a tile was not
  // issued (the end is near: then everything has to land)
  bool flowing = true;
  nxt = cur;
  enter();
  for (int q = 0; q < S; ++q) flowing &= issue(lds0 + q * (BUF * 2));
  if (flowing) tile_barrier_but<(S - 1) * NQ>();
  else tile_barrier();
#pragma unroll
  for (int f = 0; f < NF; ++f) read(f, 0, 0);
  uint32_t lq = lds0;  // the buffer being read, where the next copies go
  const uint32_t lds_last = lds0 + (S - 1) * (BUF * 2);
  int landed = 0;      // that many tiles were waited for ahead of an epilogue

  auto first_half = [&](uint32_t hop) {
    unroll<B4>([&](auto B) {
      constexpr int b = B.value, x = b / PR * 4, i = x / MI, j = x % MI, pn_ = b % PR == 1 ? 1 : 0, pm_ = b % PR == 2 ? 1 : 0;
#pragma unroll
      for (int f = ahead(b); f < ahead(b + 1); ++f) read(f, 1, 1);
      if constexpr (MI == 2)
        mfma2x2(acc[0][0], acc[0][1], acc[1][0], acc[1][1], fn[0][pn_][0], fn[0][pn_][1], fm[0][pm_][0], fm[0][pm_][1]);
      else
        mfma4<BIG>(acc[i][j], acc[i][j + 1], acc[i][j + 2], acc[i][j + 3], fn[0][pn_][i], fm[0][pm_][j], fm[0][pm_][j + 1],
                   fm[0][pm_][j + 2], fm[0][pm_][j + 3]);
      if constexpr (ahead(b + 1) == NF && (b == 0 || ahead(b) < NF)) {  // the last read of this tile is out
        gm.move(hop);
        gn.move(hop);
      }
    });
  };
  // with the next k tile's copies between the MFMAs
  auto second_half = [&](uint64_t live) {
    unroll<B4>([&](auto B) {
      constexpr int b = B.value, x = b / PR * 4, i = x / MI, j = x % MI, pn_ = b % PR == 1 ? 1 : 0, pm_ = b % PR == 2 ? 1 : 0;
      // the next tile's first fragments (after the last tile: not used)
#pragma unroll
      for (int f = ahead(b); f < ahead(b + 1); ++f) read(f, 0, 0);
      // copy q: m (high, low), then n (high, low)
      auto lds_at = [](int q) constexpr {
        return q < PL * JM ? (q / JM) * (int)IMG_M + q % JM * NT * 16
                           : PL * (int)IMG_M + (q - PL * JM) / JN * (int)IMG_N + (q - PL * JM) % JN * NT * 16;
      };
      auto off_at = [&](int q) { return q < PL * JM ? sm.off[q % JM] : sn.off[(q - PL * JM < 0 ? 0 : q - PL * JM) % JN]; };
      auto base_at = [&](int q) {
        if (q < PL * JM) return q / JM ? pm2 : pm;
        const int r = q - PL * JM;
        return r / JN ? pn2 : sn.is_alt(r % JN) ? pa : pn;
      };
      constexpr int q0 = b * NQ / B4, q1 = (b + 1) * NQ / B4;
      if constexpr (MI == 2) {
        mfma2x2(acc[0][0], acc[0][1], acc[1][0], acc[1][1], fn[1][pn_][0], fn[1][pn_][1], fm[1][pm_][0], fm[1][pm_][1]);
#pragma unroll
        for (int q = q0; q < q1; ++q) dma16_if(base_at(q), off_at(q), lq + lds_at(q), live);
      } else if constexpr (q1 == q0) {
        mfma4<BIG>(acc[i][j], acc[i][j + 1], acc[i][j + 2], acc[i][j + 3], fn[1][pn_][i], fm[1][pm_][j], fm[1][pm_][j + 1],
                   fm[1][pm_][j + 2], fm[1][pm_][j + 3]);
      } else if constexpr (q1 == q0 + 1) {
        constexpr int at1 = lds_at(q0);
        mfma4_copy<BIG>(acc[i][j], acc[i][j + 1], acc[i][j + 2], acc[i][j + 3], fn[1][pn_][i], fm[1][pm_][j],
                        fm[1][pm_][j + 1], fm[1][pm_][j + 2], fm[1][pm_][j + 3], lq, live, at1, off_at(q0), base_at(q0));
      } else {
        static_assert(q1 == q0 + 2, "copies among four MFMAs");
        constexpr int at1 = lds_at(q0), at2 = lds_at(q0 + 1);
        mfma4_copy2<BIG>(acc[i][j], acc[i][j + 1], acc[i][j + 2], acc[i][j + 3], fn[1][pn_][i], fm[1][pm_][j],
                         fm[1][pm_][j + 1], fm[1][pm_][j + 2], fm[1][pm_][j + 3], lq, live, at1, off_at(q0), base_at(q0), at2,
                         off_at(q0 + 1), base_at(q0 + 1));
      }
    });
  };
  for (;;) {
    for (int n = max(1, cur.end - cur.it); n > 0; --n) {
      const uint32_t hop = S == 2 ? (lq == lds0 ? BUF * 2 : 0u - BUF * 2) : (lq == lds_last ? 0u - (S - 1) * (BUF * 2) : BUF * 2);
      first_half(hop);
      if (__builtin_expect(landed > 0, 0)) {
        tile_barrier_landed();
        --landed;
      } else if (S == 2 || __builtin_expect(!flowing, 0)) {
        tile_barrier();
      } else {
        tile_barrier_but<(S - 2) * NQ>();
      }
      const int go = run > 0 ? -1 : 0;
      if (__builtin_expect(!go, 0)) flowing &= issue(lq);  // a run's end: this k tile in one go, or nothing
      uint64_t live;  // all lanes or none, in scalar registers
      asm volatile("v_cmp_ne_u32 %0, 0, %1" : "=s"(live) : "v"(go));
      second_half(live);
      lq += hop;
      run += go;
      step_on(go);
    }
    Ctx c;
    c.m0 = cur.mt * TM + wm * WTM;
    c.n0 = cur.nt * (DUAL ? TN / 2 : TN) + wn * (DUAL ? WTN / 2 : WTN);
    c.M = M;
    c.N = cur.N;
    c.off = RAG == 2 ? g.off[cur.batch] : 0;
    c.len = RAG == 2 ? cur.N : 0;
    c.mt = cur.mt;
    c.nt = cur.nt;
    c.wm = wm;
    c.wn = wn;
    c.batch = cur.batch;
    c.split = cur.split;
    c.lane = lane;
    c.stage = lds + S * BUF + wave * STAGE;
    typename Epi::template Pre<NI, MI> pre;
    epi.load(c, pre);
    // the copies in flight land before the epilogue stores anything, so that the next barrier need
    // not wait for those stores
    copies_landed();
    landed = S - 1;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < MI; j += 4) {
        if constexpr (MI == 2) mfma_done<BIG>(acc[i][0], acc[i][1], acc[i ^ 1][0], acc[i ^ 1][1]);
        else mfma_done<BIG>(acc[i][j], acc[i][j + 1], acc[i][j + 2], acc[i][j + 3]);
      }
    epi.template run<NI, MI>(c, pre, acc);
    l_mul += hops;
    if (!tile_at<RAG, TN>(a, g, tiles_m, splits, K, l_mul, cur)) break;
    clear();
  }
}

inline int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
inline int64_t up8(int64_t x) { return (x + 7) / 8 * 8; }

// Output tiles; every shape runs four waves, two along each side. T256 and T128 double buffer (one and
// two blocks a CU); T64 keeps four buffers (two blocks a CU): for products with few tiles, whose time is
// the copies' latency.
enum { T64 = 64, T128 = 128, T256 = 256, T_ALL = T64 | T128 | T256 };
// DUAL has no 64 (its columns come in blocks of 64 of each matrix); launch_small no 256.
enum { T_DUAL = T128 | T256, T_SMALL = T64 | T128 };

template <int LM, int LN, int T, int S, bool DUAL, int RAG, int PL = 1, class Epi>
void launch_tile(Args a, Ragged g, const Epi& e, hipStream_t stream) {
  a.tiles_m = cdiv(a.M, T);
  a.tiles_n = cdiv(a.N, DUAL ? T / 2 : T);
  int64_t tiles = a.sym ? (int64_t)a.tiles_m * (a.tiles_m + 1) / 2 : (int64_t)a.tiles_m * a.tiles_n;
  tiles *= a.splits * a.batch;
  if (RAG == 2) {
    tiles = 0;
    for (int b = 0; b < g.count; ++b) {
      g.start[b] = (int)tiles;
      tiles += (int64_t)a.tiles_m * cdiv(g.len[b], T);
    }
    g.start[g.count] = (int)tiles;
  }
  const int64_t slots = (int64_t)device_cu_count() * (T > 128 || PL == 2 ? 1 : 2);  // resident blocks
  const int64_t blocks = std::min<int64_t>(tiles, slots);
  if (blocks <= 0) return;
  if constexpr (RAG != 0) gemm16_kernel<LM, LN, T, T, S, PL, DUAL, RAG, Epi><<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(a, g, e);
  else gemm16_kernel<LM, LN, T, T, S, PL, DUAL, 0, Epi><<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(a, 0, e);
}

template <int LM, int LN, bool DUAL = false, int RAG = 0, class Epi>
void launch(int tile, const Args& a, const Epi& e, hipStream_t stream, const Ragged& g = Ragged()) {
  if (tile == T256) launch_tile<LM, LN, 256, 2, DUAL, RAG>(a, g, e, stream);
  else if (DUAL || tile == T128) launch_tile<LM, LN, 128, 2, DUAL, RAG>(a, g, e, stream);
  else if constexpr (!DUAL) launch_tile<LM, LN, 64, 4, false, RAG>(a, g, e, stream);
}

// without 256x256 tiles: epilogues that need more registers than those leave
template <int LM, int LN, int RAG = 0, class Epi>
void launch_small(int tile, const Args& a, const Epi& e, hipStream_t stream, const Ragged& g = Ragged()) {
  if (tile == T64) launch_tile<LM, LN, 64, 4, false, RAG>(a, g, e, stream);
  else launch_tile<LM, LN, 128, 2, false, RAG>(a, g, e, stream);
}

// Split values (PL 2): one block a CU at either tile. A k tile, with its three products, takes 1.27 us at
// 128x128 and 0.42 at 64x64, a tile's end 5.7 and 3 (K = 512 to 2048).
inline int plan_split(int64_t tiles128, int64_t tiles64, int64_t K) {
  const int cus = device_cu_count();
  const double kt = cdiv(K, BK);
  const double t128 = cdiv(tiles128, cus) * (kt * 1.27 + 5.7), t64 = cdiv(tiles64, cus) * (kt * 0.42 + 3.0);
  return t64 < t128 ? T64 : T128;
}
template <int LM, int LN, int RAG = 0, class Epi>
void launch_split(int tile, const Args& a, const Epi& e, hipStream_t stream, const Ragged& g = Ragged()) {
  if (tile == T64) launch_tile<LM, LN, 64, 4, false, RAG, 2>(a, g, e, stream);
  else launch_tile<LM, LN, 128, 2, false, RAG, 2>(a, g, e, stream);
}

// How to run a product: the tile and the k splits with the least estimated time, in us. Measured on
// MI355X (16-bit operands, K = 768 and more): a 64-wide k tile takes 1.45 at 256x256; at 128x128 0.67 with
// one block on a CU and 0.93 with two; at 64x64 0.3 and 0.57. A tile's end costs about 7, 4 and 1.5
// more (`epi` scales it for epilogues that compute), a launch 4; splits pay a second launch and their
// slabs' way through memory at 4 TB/s. `allowed`: the tiles that
// the launch has.
struct Plan {
  int tile, splits;
};
inline Plan plan(int64_t M, int64_t N, int64_t K, int nseg, int batch, bool sym, bool may_split, double epi = 1.0,
                 int allowed = T_ALL) {
  Plan best{T128, 1};
  double best_t = 1e30;
  const int64_t kt = (int64_t)cdiv(K, BK) * nseg;
  const int cus = device_cu_count();
  for (int tile : {T256, T128, T64}) {
    if (!(allowed & tile)) continue;
    const int64_t tm = cdiv(M, tile), tn = cdiv(N, tile);
    const int64_t tiles = (sym ? tm * (tm + 1) / 2 : tm * tn) * batch;
    for (int s = 1; s <= 64 && (s == 1 || (may_split && kt / s >= 4)); ++s) {
      const bool two = tile != T256 && tiles * s > cus;  // blocks on a CU
      const int64_t slots = two ? 2 * cus : cus;
      const double unit = tile == T256 ? 1.45 : tile == T128 ? (two ? 0.93 : 0.67) : (two ? 0.57 : 0.3);
      const double end = epi * (tile == T256 ? 7.0 : tile == T128 ? 4.0 : 1.5);
      const double rounds = (double)((tiles * s + slots - 1) / slots);
      double t = 4.0 + rounds * ((double)((kt + s - 1) / s) * unit + end);
      if (s > 1) t += 4.0 + (double)M * N * batch * (s + 0.5) * 8.0 / 4e6;
      if (t < best_t) {
        best_t = t;
        best = {tile, s};
      }
    }
  }
  return best;
}

// The rule that plan()'s terms give a product with a device count of at most M rows.
inline SplitRule split_rule(int64_t M, int64_t N, int64_t K, const Plan& p, int* chosen) {
  SplitRule r;
  r.chosen = chosen;
  r.tile = p.tile;
  r.tn = cdiv(N, p.tile);
  r.kt = cdiv(K, BK);
  r.cus = device_cu_count();
  r.unit1 = p.tile == T256 ? 145 : p.tile == T128 ? 67 : 30;
  r.unit2 = p.tile == T256 ? 0 : p.tile == T128 ? 93 : 57;
  r.end = p.tile == T256 ? 700 : p.tile == T128 ? 400 : 150;
  r.N = (int)N;
  r.cap = std::max(cdiv(M, p.tile) * p.splits, cdiv((p.tile == T256 ? 1 : 2) * r.cus, r.tn));
  return r;
}

// ---- epilogues -----------------------------------------------------------------------------
// An epilogue is a struct with `load` (what it reads from memory early, into a Pre: on its way while
// the tile's copies land) and `run` (its work on the accumulators: acc[i][j][k] is column
// n0 + 16 i + 4 (lane >> 4) + k of row m0 + 16 j + (lane & 15)).
// ---- helpers ---------------------------------------------------------------------- //
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

// Eight consecutive values of a row: one 16-byte store when `vec` (rows start 16-byte aligned).
__device__ __forceinline__ void store8(u16* row, int n, int N, bool vec, uint4 v) {
  if (vec && n + 7 < N) {
    *reinterpret_cast<uint4*>(row + n) = v;
    return;
  }
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (n + k < N) row[n + k] = (u16)(w[k >> 1] >> (16 * (k & 1)));
}

// A factor that lives on the device: *f, or 1, over an optional count (0 if that is 0).
__device__ __forceinline__ float scalar(const float* f, const int* count) {
  const float v = f ? *f : 1.f;
  if (!count) return v;
  return *count > 0 ? v / (float)*count : 0.f;
}

// out[batch][m][n] = alpha * acc, rounded once to the 16-bit format; alpha times an optional device
// scalar over an optional device count. `out[]` holds one base per batch entry.
struct EpiStore {
  u16* out[2];
  int64_t ld;
  float alpha;
  const float* dev_alpha;
  const int* dev_count;
  template <int NI, int MI>
  struct Pre {};
  template <int NI, int MI>
  __device__ __forceinline__ void load(const Ctx&, Pre<NI, MI>&) const {}
  template <int NI, int MI>
  __device__ __forceinline__ void run(const Ctx& c, const Pre<NI, MI>&, f32x4 (&acc)[NI][MI]) const {
    const float al = alpha * scalar(dev_alpha, dev_count);
    u16* o = c.batch == 0 ? out[0] : out[1];
    const bool vec = (ld & 7) == 0;
    const RowStage<NI * 16> st{c.stage, c.lane};
#pragma unroll
    for (int j = 0; j < MI; ++j) {
      pin(acc, j);
#pragma unroll
      for (int i = 0; i < NI; ++i)
        st.put(i, pack4bf(acc[i][j][0] * al, acc[i][j][1] * al, acc[i][j][2] * al, acc[i][j][3] * al));
      st.turn();
#pragma unroll
      for (int g = 0; g < st.GETS; ++g) {
        const int m = c.m0 + j * 16 + st.row(g);
        const uint4 v = st.get(g);
        if (m < c.M) store8(o + (int64_t)m * ld, c.n0 + st.col(), c.N, vec, v);
      }
      st.turn();
    }
  }
};

// fp32 slab of one k split: slab[batch * splits + split][m][n] (+)= acc. ld is a multiple of 4. With a stride
// of 0 the slabs are as long as the device's count of rows.
struct EpiSlab {
  float* slab;
  int64_t ld, stride;
  int splits, add;
  template <int NI, int MI>
  struct Pre {};
  template <int NI, int MI>
  __device__ __forceinline__ void load(const Ctx&, Pre<NI, MI>&) const {}
  template <int NI, int MI>
  __device__ __forceinline__ void run(const Ctx& c, const Pre<NI, MI>&, f32x4 (&acc)[NI][MI]) const {
    float* o = slab + (int64_t)(c.batch * splits + c.split) * (stride ? stride : c.M * ld);
#pragma unroll
    for (int j = 0; j < MI; ++j) {
      const int m = c.m0 + j * 16 + (c.lane & 15);
      pin(acc, j);
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

// out[batch][m][n] = sum of the slabs, in split order
static __global__ void __launch_bounds__(256) slab_sum(const float* __restrict__ slab, int splits, int64_t stride,
                                                       int64_t ld, int M, int N, u16* __restrict__ out0,
                                                       u16* __restrict__ out1, int64_t ldo) {
  const int n4 = (N + 3) >> 2;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t m = i / n4;
  const int n = (int)(i - m * n4) * 4;
  if (m >= M) return;
  const float* p = slab + (int64_t)blockIdx.y * splits * stride + m * ld + n;
  f32x4 s = *reinterpret_cast<const f32x4*>(p);
  for (int q = 1; q < splits; ++q) s += *reinterpret_cast<const f32x4*>(p + q * stride);
  store4((blockIdx.y ? out1 : out0) + m * ldo, n, N, (ldo & 3) == 0, s[0], s[1], s[2], s[3]);
}

// A product rounded once into 16-bit outputs (one or two batch entries), split along k when its
// tiles alone leave CUs idle.
inline Plan product_plan(int64_t M, int64_t N, int64_t K, int nseg = 1, int batch = 1) {
  return plan(M, N, K, nseg, batch, false, true);
}
template <int LM, int LN>
void product(Args a, u16* out0, u16* out1, int64_t ldo, c10::Device dev, hipStream_t stream) {
  const Plan p = product_plan(a.M, a.N, a.K, a.nseg, a.batch);
  a.splits = p.splits;
  if (p.splits == 1) {
    launch<LM, LN>(p.tile, a, EpiStore{{out0, out1}, ldo, 1.f, nullptr, nullptr}, stream);
    return;
  }
  const int64_t ld = up8(a.N), stride = (int64_t)a.M * ld;
  at::Tensor slab = at::empty({a.batch * a.splits * stride}, at::TensorOptions().device(dev).dtype(at::kFloat));
  launch<LM, LN>(p.tile, a, EpiSlab{slab.data_ptr<float>(), ld, stride, a.splits, 0}, stream);
  slab_sum<<<dim3(cdiv((int64_t)a.M * ((a.N + 3) / 4), 256), a.batch), 256, 0, stream>>>(
      slab.data_ptr<float>(), a.splits, stride, ld, a.M, a.N, out0, out1, ldo);
}

}  // namespace g16
MIHVD_OPNS_END
