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
  int chunk;        // rows whose labels are counted ahead, or 0: each block counts for itself
};
constexpr int LCE_BLOCKS = 256;  // that share the end of the forward pass: partial sums of the loss
// The labelled rows: compact position -> row, row -> compact position or -1, their labels and count.
struct LceRows {
  const int* idx;
  const int* inv;
  const int* label;
  const int* cnt;
};
struct LceRowsOut {
  int *idx, *inv, *label, *cnt;
  int* done;    // blocks of the last kernel that have ended
  int* counts;  // labelled rows per chunk
};
struct LceGrad {
  const float* scale;     // G, one device scalar
  const int* div;         // what it is divided by (the mean's count), or null
  const float* rowscale;  // g_r / G per compact row, or null
};
struct LceScratch {
  int piece;     // vocabulary entries per piece
  int64_t ldz;   // row stride of dz, a multiple of 8
  u16* dz;       // [N][ldz]
  float* dbp;    // [2 * tiles of rows][ldz]
  int splits, dz_tile, dh_tile, dw_tile;
  int64_t slab_rows;  // that the splits of dh need at any count of labelled rows
  float* slab;        // [slab_rows][K8]
  int* chosen;        // the splits that the device chose
};

// How the products of a shape run (tiles, k splits of the hidden gradient); x.piece is set.
void lce_plan(LceShape& s);
void lce_plan_backward(LceShape& s, LceScratch& x, bool bias);

#define MIHVD_TRANSFORMER_DECLS                                                                                        \
  void lce_forward_16(const LceShape& s, const int64_t* labels, int64_t ignore, const LceRowsOut& rw, const u16* h,      \
                      int64_t hs0, int64_t hs1, const u16* w, int64_t ldw, const void* bias, int bias_kind, u16* hc,   \
                      float2* part, float* zlab, float2* lse, float* rows, float* blocks, float* loss, int mean,       \
                      hipStream_t st);                                                                                 \
  void lce_backward_16(const LceShape& s, const LceRows& rw, const LceGrad& g, const u16* hc, const u16* w,            \
                       int64_t ldw, const void* bias, int bias_kind, const float2* lse, const LceScratch& x, u16* dh,  \
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

// Tiles and k splits: the gate product (0: the kernels for few rows); y, dWd, the batch of dWg and dWu, dx.
struct FfnPlan {
  int gate, tile[4], splits[4];
};
FfnPlan ffn_plan(const FfnShape& s);

MIHVD_TRANSFORMER_DECLS
namespace f16 {
MIHVD_TRANSFORMER_DECLS
}

// Newton-Schulz (newton_schulz.hip): matrices whose smaller sides are alike, padded to the products' k
// tile of 64. X of each is held with the smaller side as rows: [planes][side][len], one matrix behind the
// other.
constexpr int NS_MAX = 32;
struct NsMat {
  const void* src;  // the matrix (orthogonalize) / gradient (Muon), [rows][cols]
  void* dst;        // result / weight
  float* mom;       // Muon: momentum
  int rows, cols, len;
  int64_t off;      // of X, in elements
  float step;       // Muon: lr * scale
};
struct NsGroup {
  int count, side;
  int planes;  // 1: fp16; 2: fp16 hi + lo
  NsMat m[NS_MAX];
};
struct NsParams {
  int steps;
  float a, b, c, eps;
  int src_kind;  // 0 fp32, 1 bf16, 2 fp16
  int muon, nesterov;
  float momentum, decay;  // p = p * decay - step * O
};
struct NsScratch {
  u16 *x0, *x1;       // X before and after a step
  u16 *gram, *poly;   // [count][planes][side][side]
  double* partial;    // [count][NS_PART]
};
constexpr int NS_PART = 64;
struct NsPlan {
  int gram, poly, update, last;
};
NsPlan ns_plan(const NsGroup& g);
void ns_run(const NsGroup& g, const NsParams& p, const NsScratch& s, hipStream_t st);

}  // namespace mihvd
