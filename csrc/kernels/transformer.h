// Interfaces between transformer_ops.cpp (checks, workspaces, registration) and the kernels that are
// compiled once per 16-bit operand format (linear_ce.hip, gated_ffn.hip) or for fp16 operands only
// (newton_schulz.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <c10/core/Device.h>

namespace mihvd {

typedef unsigned short u16;

struct LceShape {
  int N, K, K8, V;  // rows, hidden size, hidden size padded to 8, vocabulary
  int tile, npart;  // of the logits: output tile, (max, sum) pairs per row (two waves along a tile)
};
// The labelled rows: compact position -> row, row -> compact position or -1, their labels and count.
struct LceRows {
  const int* idx;
  const int* inv;
  const int* label;
  const int* cnt;
};
struct LceGrad {
  const float* scale;     // G (times 1 / count for the mean), one device scalar
  const float* rowscale;  // g_r / G per compact row, or null
};
struct LceScratch {
  int piece;     // vocabulary entries per piece
  int64_t ldz;   // row stride of dz, a multiple of 8
  u16* dz;       // [N][ldz]
  float* dbp;    // [2 * tiles of rows][ldz]
  int splits, dh_tile, dw_tile;
  float* slab;   // [splits][N][K8]
};

// How the products of a shape run (tiles, k splits of the hidden gradient); x.piece is set.
void lce_plan(LceShape& s);
void lce_plan_backward(LceShape& s, LceScratch& x);

#define MIHVD_TRANSFORMER_DECLS                                                                                        \
  void lce_forward_16(const LceShape& s, const LceRows& rw, const u16* h, int64_t hs0, int64_t hs1, const u16* w,      \
                      int64_t ldw, const void* bias, int bias_kind, u16* hc, float2* part, float* zlab, float* lse,    \
                      float* rows, float* loss, int mean, hipStream_t st);                                             \
  void lce_backward_16(const LceShape& s, const LceRows& rw, const LceGrad& g, const u16* hc, const u16* w,            \
                       int64_t ldw, const void* bias, int bias_kind, const float* lse, const LceScratch& x, u16* dh,   \
                       u16* dw, void* db, hipStream_t st);                                                             \
  void ffn_forward_16(const FfnShape& s, const u16* x, int64_t ldx, const FfnWeights& w, int act, u16* g, u16* u,        \
                      u16* h, u16* y, c10::Device dev, hipStream_t st);                                                \
  void ffn_backward_16(const FfnShape& s, const u16* dy, int64_t lddy, const u16* x, int64_t ldx, const FfnWeights& w, \
                       int act, const u16* g, const u16* u, const u16* h, u16* dgu, u16* dx, u16* dwg, u16* dwu,       \
                       u16* dwd, c10::Device dev, hipStream_t st);

struct FfnShape {
  int N, K, K8, F, F8;
};
// w_gate [F][ldg], w_up [F][ldu] (one leading dimension for both), w_down [K][ldd]
struct FfnWeights {
  const u16 *gate, *up, *down;
  int64_t ldgu, ldd;
};
enum { ACT_SILU = 0, ACT_GELU, ACT_GELU_TANH, ACT_RELU, ACT_SIGMOID, ACT_COUNT };

MIHVD_TRANSFORMER_DECLS
namespace f16 {
MIHVD_TRANSFORMER_DECLS
}

// Newton-Schulz (newton_schulz.hip): one group of equally shaped matrices.
constexpr int NS_MAX = 32;
struct NsGroup {
  int count, rows, cols;
  int rp, cp, sp;  // rows, cols and the smaller of them, padded to the products' k tile of 64
  int planes;                           // 1: fp16; 2: fp16 hi + lo
  const void* src[NS_MAX];              // u (orthogonalize) / gradient (Muon)
  void* dst[NS_MAX];                    // result / weight
  float* mom[NS_MAX];                   // Muon: momentum
};
struct NsParams {
  int steps;
  float a, b, c, eps;
  int src_kind;  // 0 fp32, 1 bf16, 2 fp16
  int muon;
  float lr, momentum, decay, scale;  // p = p * decay - lr * scale * O
  int nesterov;
};
struct NsScratch {
  u16 *x0, *x1, *gram, *poly;  // planes: [count][planes][...]
  float* partial;              // [count][NS_PART]
};
constexpr int NS_PART = 64;
void ns_run(const NsGroup& g, const NsParams& p, const NsScratch& s, hipStream_t st);

}  // namespace mihvd
