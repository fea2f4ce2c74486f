// torch.ops.mihvd registration of the transformer-step operators: argument checks, packing of
// operands the matrix core cannot read in place, workspaces, and the choice of the operand format.
#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/variable.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/library.h>

#include <initializer_list>
#include <map>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "common.h"
#include "transformer.h"

namespace mihvd {
namespace {

constexpr int64_t MAX_ROWS = int64_t(1) << 30, MAX_LD = int64_t(1) << 22;
constexpr int64_t LCE_CHUNKS = 4096;
constexpr int64_t DZ_BYTES = int64_t(512) << 20;  // bound on the gradient piece that backward holds

inline int64_t up8(int64_t x) { return (x + 7) / 8 * 8; }
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline hipStream_t cur_stream() { return c10::hip::getCurrentHIPStream().stream(); }

const u16* p16(const at::Tensor& t) { return static_cast<const u16*>(t.data_ptr()); }
u16* m16(at::Tensor& t) { return t.defined() ? static_cast<u16*>(t.data_ptr()) : nullptr; }

// [R][C] with any strides -> [R][C8], the padding zero
__global__ void __launch_bounds__(256) pack_kernel(const u16* __restrict__ src, int64_t s0, int64_t s1, int64_t R, int C,
                                                   int C8, u16* __restrict__ dst) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < R * C8; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / C8;
    const int c = (int)(i - r * C8);
    dst[i] = c < C ? src[r * s0 + c * s1] : (u16)0;
  }
}

// A matrix the core reads: rows of unit stride, 16-byte aligned, columns a multiple of 8; anything
// else is copied into that form once.
struct Mat {
  at::Tensor hold;
  const u16* p;
  int64_t ld;
};
bool direct(const at::Tensor& t) {
  return t.stride(1) == 1 && t.size(1) % 8 == 0 && t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) &&
         t.stride(0) <= MAX_LD && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}
Mat mat(const at::Tensor& t, bool force = false) {
  if (!force && direct(t)) return {t, p16(t), t.stride(0)};
  const int64_t R = t.size(0), C = t.size(1), C8 = up8(C);
  at::Tensor d = at::empty({R, C8}, t.options());
  const int64_t blocks = std::min<int64_t>(cdiv(R * C8, 256), 8192);
  if (blocks > 0)
    pack_kernel<<<dim3((unsigned)blocks), 256, 0, cur_stream()>>>(p16(t), t.stride(0), t.stride(1), R, (int)C, (int)C8,
                                                                  m16(d));
  return {d, p16(d), C8};
}

void check16(const at::Tensor& t, const char* op, const char* name, const at::Tensor& like, int64_t dim) {
  TORCH_CHECK_VALUE(t.dim() == dim, op, ": ", name, " must have ", dim, " dimensions (got ", t.dim(), ")");
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, op, ": ", name,
                   " must be bfloat16 or float16 (float32 under autocast; got ", t.scalar_type(), ")");
  TORCH_CHECK_TYPE(t.scalar_type() == like.scalar_type(), op, ": ", name, " must have the type of the first argument");
  TORCH_CHECK_VALUE(t.device() == like.device() && t.is_cuda(), op, ": ", name, " must be on the same GPU");
}

// ------------------------------------------------------------------------------------------ //
// linear_cross_entropy

// Row weights: G = max |g_r| over the finite ones (an infinite one stays infinite in its own row), g_r / G.
__global__ void __launch_bounds__(1024) lce_scale(const float* __restrict__ gout, int64_t gstride,
                                                  const int* __restrict__ idx, const int* __restrict__ cnt,
                                                  float* __restrict__ scale, float* __restrict__ rowscale) {
  const int n = *cnt;
  __shared__ float sh[16];
  float m = 0.f;
  for (int c = threadIdx.x; c < n; c += 1024) {
    const float g = fabsf(gout[idx[c] * gstride]);
    if (g < INFINITY) m = fmaxf(m, g);
  }
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = m;
  __syncthreads();
  m = sh[0];
  for (int i = 1; i < 16; ++i) m = fmaxf(m, sh[i]);
  const float G = m > 0.f ? m : 1.f;
  for (int c = threadIdx.x; c < n; c += 1024) rowscale[c] = gout[idx[c] * gstride] / G;
  if (threadIdx.x == 0) *scale = G;
}

// meta: row numbers, places, labels, their count, and the forward pass's block counter and chunk counts
LceRows rows_of(const at::Tensor& meta, int64_t N) {
  const int* p = meta.data_ptr<int>();
  return {p, p + N, p + 2 * N, p + 3 * N};
}
int bias_kind(const c10::optional<at::Tensor>& b) { return !b ? 0 : b->scalar_type() == at::kFloat ? 1 : 2; }

void lce_check(const at::Tensor& h, const at::Tensor& w, const c10::optional<at::Tensor>& bias) {
  const char* op = "linear_cross_entropy";
  check16(h, op, "hidden", h, 2);
  check16(w, op, "weight", h, 2);
  const int64_t N = h.size(0), K = h.size(1), V = w.size(0);
  TORCH_CHECK_VALUE(w.size(1) == K, op, ": weight has ", w.size(1), " columns, hidden has ", K);
  TORCH_CHECK_VALUE(K >= 1 && V >= 1 && N <= MAX_ROWS && V <= MAX_ROWS && K <= MAX_LD, op, ": sizes out of range (",
                    N, " rows, ", K, " hidden, ", V, " vocabulary)");
  if (bias) {
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == V && bias->device() == h.device(), op,
                      ": bias must be a vector of ", V, " on the same GPU");
    TORCH_CHECK_TYPE(bias->scalar_type() == at::kFloat || bias->scalar_type() == h.scalar_type(), op,
                     ": bias must be float32 or of hidden's type");
  }
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> lce_forward(const at::Tensor& h, const at::Tensor& w,
                                                                       const at::Tensor& labels,
                                                                       const c10::optional<at::Tensor>& bias_in,
                                                                       int64_t ignore_index, int64_t reduction) {
  lce_check(h, w, bias_in);
  const int64_t N = h.size(0), K = h.size(1), V = w.size(0), K8 = up8(K);
  TORCH_CHECK_TYPE(labels.scalar_type() == at::kLong, "linear_cross_entropy: labels must be int64");
  TORCH_CHECK_VALUE(labels.dim() == 1 && labels.size(0) == N && labels.device() == h.device(),
                    "linear_cross_entropy: labels must be a vector of ", N, " on the same GPU");
  TORCH_CHECK_VALUE(reduction >= 0 && reduction <= 2, "linear_cross_entropy: reduction");
  c10::DeviceGuard guard(h.device());
  hipStream_t st = cur_stream();
  const auto f32 = h.options().dtype(at::kFloat);
  c10::optional<at::Tensor> bias;
  if (bias_in) bias = bias_in->contiguous();
  LceShape s{(int)N, (int)K, (int)K8, (int)V, 0, 0, 0};
  // Blocks that count all labels ahead of their rows for themselves read 64 KB on average at 16384 rows; past that
  // the chunks (at most LCE_CHUNKS) are counted ahead, which costs a launch.
  if (N > 16384) s.chunk = (int)(cdiv(cdiv(N, LCE_CHUNKS), 1024) * 1024);
  at::Tensor loss = reduction ? at::empty({}, f32) : at::empty({N}, f32);
  at::Tensor hc = at::empty({N, K8}, h.options()), lse = at::empty({N, 2}, f32);
  at::Tensor meta = at::empty({3 * N + 2 + LCE_CHUNKS}, h.options().dtype(at::kInt));
  if (N == 0) {
    if (reduction) loss.fill_(reduction == 1 ? NAN : 0.f);
    meta.zero_();
    return {loss, hc, meta, lse};
  }
  const at::Tensor lab = labels.contiguous();
  int* m = meta.data_ptr<int>();
  const LceRowsOut rw{m, m + N, m + 2 * N, m + 3 * N, m + 3 * N + 1, m + 3 * N + 2};
  const Mat wm = mat(w);
  lce_plan(s);
  // (max, sum) pairs, the labels' logits, the blocks' sums
  at::Tensor work = at::empty({N * (2 * (int64_t)s.npart + 1) + LCE_BLOCKS}, f32);
  float* part = work.data_ptr<float>();
  float *zlab = part + 2 * N * s.npart, *blocks = zlab + N;
  auto run = h.scalar_type() == at::kHalf ? &f16::lce_forward_16 : &lce_forward_16;
  run(s, lab.data_ptr<int64_t>(), ignore_index, rw, p16(h), h.stride(0), h.stride(1), wm.p, wm.ld,
      bias ? bias->data_ptr() : nullptr, bias_kind(bias), m16(hc), reinterpret_cast<float2*>(part), zlab,
      reinterpret_cast<float2*>(lse.data_ptr<float>()), reduction ? nullptr : loss.data_ptr<float>(), blocks,
      reduction ? loss.data_ptr<float>() : nullptr, reduction == 1, st);
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {loss, hc, meta, lse};
}

void lce_pieces(const LceShape& s, LceScratch& x) {
  const int64_t N = s.N;
  x.piece = (int)std::min<int64_t>(up8(s.V), std::max<int64_t>(256, DZ_BYTES / (2 * N) / 256 * 256));
  x.ldz = up8(x.piece);
}

// The gradients that are asked for, in the order hidden, weight, bias.
std::vector<at::Tensor> wanted(std::initializer_list<at::Tensor> ts) {
  std::vector<at::Tensor> r;
  for (const at::Tensor& t : ts)
    if (t.defined()) r.push_back(t);
  return r;
}
std::vector<at::Tensor> lce_backward(const at::Tensor& gout, const at::Tensor& hc, const at::Tensor& w,
                                     const c10::optional<at::Tensor>& bias_in, const at::Tensor& meta, const at::Tensor& lse,
                                     int64_t reduction, bool need_h, bool need_w, bool need_b) {
  const int64_t N = lse.size(0), V = w.size(0), K = w.size(1), K8 = up8(K);
  TORCH_CHECK_VALUE(hc.dim() == 2 && hc.size(0) == N && hc.size(1) == K8 && hc.is_contiguous() &&
                        meta.numel() >= 3 * N + 2 && hc.scalar_type() == w.scalar_type(),
                    "lce_backward: not the tensors that lce_forward returned");
  check16(w, "lce_backward", "weight", hc, 2);
  TORCH_CHECK_VALUE(gout.scalar_type() == at::kFloat && gout.device() == w.device() &&
                        (reduction ? gout.numel() == 1 : (gout.dim() == 1 && gout.size(0) == N)),
                    "lce_backward: the loss gradient does not fit the loss");
  c10::DeviceGuard guard(w.device());
  hipStream_t st = cur_stream();
  const auto f32 = w.options().dtype(at::kFloat);
  c10::optional<at::Tensor> bias;
  if (bias_in) bias = bias_in->contiguous();
  need_b = need_b && bias.has_value();
  at::Tensor dh, dw, db;
  if (need_h) dh = at::empty({N, K}, w.options());
  if (need_w) dw = at::empty({V, K}, w.options());
  if (need_b) db = at::empty({V}, bias->options());
  if (N == 0) {
    if (need_w) dw.zero_();
    if (need_b) db.zero_();
    return wanted({dh, dw, db});
  }
  const LceRows rw = rows_of(meta, N);
  LceGrad g{gout.data_ptr<float>(), reduction == 1 ? rw.cnt : nullptr, nullptr};
  at::Tensor scale;
  if (reduction == 0) {
    scale = at::empty({N + 1}, f32);
    float* q = scale.data_ptr<float>();
    lce_scale<<<1, 1024, 0, st>>>(gout.data_ptr<float>(), gout.stride(0), rw.idx, rw.cnt, q, q + 1);
    g = {q, nullptr, q + 1};
  }
  const Mat wm = mat(w);
  LceScratch x{};
  LceShape s{(int)N, (int)K, (int)K8, (int)V, 0, 0, 0};
  lce_pieces(s, x);
  lce_plan_backward(s, x, bias.has_value());
  at::Tensor dz = at::empty({N, x.ldz}, w.options()), dbp, slab;
  x.dz = m16(dz);
  if (bias) {
    dbp = at::empty({2 * cdiv(N, x.dz_tile), x.ldz}, f32);
    x.dbp = dbp.data_ptr<float>();
  }
  if (need_h) {
    slab = at::empty({x.slab_rows * K8 + 1}, f32);
    x.slab = slab.data_ptr<float>();
    x.chosen = reinterpret_cast<int*>(x.slab + x.slab_rows * K8);
  }
  auto run = w.scalar_type() == at::kHalf ? &f16::lce_backward_16 : &lce_backward_16;
  run(s, rw, g, p16(hc), wm.p, wm.ld, bias ? bias->data_ptr() : nullptr, bias_kind(bias),
      reinterpret_cast<const float2*>(lse.data_ptr<float>()), x, m16(dh), m16(dw), need_b ? db.data_ptr() : nullptr, st);
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return wanted({dh, dw, db});
}

// ------------------------------------------------------------------------------------------ //
// gated_ffn

struct FfnMats {
  Mat gate, up, down;
  FfnWeights w;
};
FfnMats ffn_weights(const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd) {
  // one leading dimension serves both input projections
  const bool same = direct(wg) && direct(wu) && wg.stride(0) == wu.stride(0);
  FfnMats m{mat(wg, !same), mat(wu, !same), mat(wd), {}};
  m.w = {m.gate.p, m.up.p, m.down.p, m.gate.ld, m.down.ld};
  return m;
}
void ffn_check(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t act) {
  const char* op = "gated_ffn";
  check16(x, op, "x", x, 2);
  check16(wg, op, "w_gate", x, 2);
  check16(wu, op, "w_up", x, 2);
  check16(wd, op, "w_down", x, 2);
  const int64_t N = x.size(0), K = x.size(1), F = wg.size(0);
  TORCH_CHECK_VALUE(wg.size(1) == K && wu.size(0) == F && wu.size(1) == K && wd.size(0) == K && wd.size(1) == F, op,
                    ": w_gate and w_up must be [inner, ", K, "] and w_down [", K, ", inner]");
  TORCH_CHECK_VALUE(N <= MAX_ROWS && K >= 1 && F >= 1 && K <= MAX_LD && F <= MAX_LD / 2, op, ": sizes out of range (", N,
                    " rows, ", K, " hidden, ", F, " inner)");
  TORCH_CHECK_VALUE(act >= 0 && act < ACT_COUNT, op, ": unknown activation");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> ffn_forward(const at::Tensor& x, const at::Tensor& wg,
                                                                       const at::Tensor& wu, const at::Tensor& wd,
                                                                       int64_t act, bool save) {
  ffn_check(x, wg, wu, wd, act);
  c10::DeviceGuard guard(x.device());
  const int64_t N = x.size(0), K = x.size(1), F = wg.size(0), F8 = up8(F);
  at::Tensor y = at::empty({N, K}, x.options()), h = at::empty({N, F8}, x.options());
  at::Tensor g, u;
  if (save) {
    g = at::empty({N, F8}, x.options());
    u = at::empty({N, F8}, x.options());
  }
  if (N > 0) {
    const Mat xm = mat(x);
    const FfnMats wm = ffn_weights(wg, wu, wd);
    const FfnShape s{(int)N, (int)K, (int)up8(K), (int)F, (int)F8};
    auto run = x.scalar_type() == at::kHalf ? &f16::ffn_forward_16 : &ffn_forward_16;
    run(s, xm.p, xm.ld, wm.w, (int)act, m16(g), m16(u), m16(h), m16(y), x.device(), cur_stream());
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return {y, g, u, h};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> ffn_train(const at::Tensor& x, const at::Tensor& wg,
                                                                     const at::Tensor& wu, const at::Tensor& wd, int64_t act) {
  return ffn_forward(x, wg, wu, wd, act, true);
}
at::Tensor ffn_infer(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t act) {
  return std::get<0>(ffn_forward(x, wg, wu, wd, act, false));
}

std::vector<at::Tensor> ffn_backward(
    const at::Tensor& dy, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd,
    const at::Tensor& g, const at::Tensor& u, const at::Tensor& h, int64_t act, bool need_x, bool need_g, bool need_u,
    bool need_d) {
  ffn_check(x, wg, wu, wd, act);
  const int64_t N = x.size(0), K = x.size(1), F = wg.size(0), F8 = up8(F);
  check16(dy, "gated_ffn", "the output gradient", x, 2);
  TORCH_CHECK_VALUE(dy.size(0) == N && dy.size(1) == K, "gated_ffn: the output gradient's shape");
  for (const at::Tensor* t : {&g, &u, &h})
    TORCH_CHECK_VALUE(t->dim() == 2 && t->size(0) == N && t->size(1) == F8 && t->is_contiguous() &&
                          t->scalar_type() == x.scalar_type() && t->device() == x.device(),
                      "gated_ffn: not the tensors that the forward pass kept");
  c10::DeviceGuard guard(x.device());
  at::Tensor dx, dwg, dwu, dwd;
  if (need_x) dx = at::empty({N, K}, x.options());
  if (need_g) dwg = at::empty({F, K}, x.options());
  if (need_u) dwu = at::empty({F, K}, x.options());
  if (need_d) dwd = at::empty({K, F}, x.options());
  if (N == 0) {
    for (at::Tensor* t : {&dwg, &dwu, &dwd})
      if (t->defined()) t->zero_();
    return wanted({dx, dwg, dwu, dwd});
  }
  at::Tensor dgu;
  if (need_x || need_g || need_u) dgu = at::empty({N, 2 * F8}, x.options());
  const Mat xm = mat(x), dym = mat(dy);
  const FfnMats wm = ffn_weights(wg, wu, wd);
  const FfnShape s{(int)N, (int)K, (int)up8(K), (int)F, (int)F8};
  auto run = x.scalar_type() == at::kHalf ? &f16::ffn_backward_16 : &ffn_backward_16;
  run(s, dym.p, dym.ld, xm.p, xm.ld, wm.w, (int)act, p16(g), p16(u), p16(h), m16(dgu), m16(dx), m16(dwg), m16(dwu),
      m16(dwd), x.device(), cur_stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return wanted({dx, dwg, dwu, dwd});
}

// ------------------------------------------------------------------------------------------ //
// Shapes and types alone, for tensors without data (tracing): the checks are the kernels' own.

c10::SymInt sym8(const c10::SymInt& n) { return (n + 7) / 8 * 8; }

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> lce_forward_meta(const at::Tensor& h, const at::Tensor&,
                                                                            const at::Tensor&, const c10::optional<at::Tensor>&,
                                                                            int64_t, int64_t reduction) {
  const c10::SymInt N = h.sym_size(0);
  const auto f32 = h.options().dtype(at::kFloat);
  return {reduction ? at::empty({}, f32) : at::empty_symint({N}, f32), at::empty_symint({N, sym8(h.sym_size(1))}, h.options()),
          at::empty_symint({N * 3 + (2 + LCE_CHUNKS)}, h.options().dtype(at::kInt)), at::empty_symint({N, 2}, f32)};
}
std::vector<at::Tensor> lce_backward_meta(const at::Tensor&, const at::Tensor& hc, const at::Tensor& w,
                                          const c10::optional<at::Tensor>& bias, const at::Tensor&, const at::Tensor&, int64_t,
                                          bool need_h, bool need_w, bool need_b) {
  at::Tensor dh, dw, db;
  if (need_h) dh = at::empty_symint({hc.sym_size(0), w.sym_size(1)}, w.options());
  if (need_w) dw = at::empty_symint(w.sym_sizes(), w.options());
  if (need_b && bias) db = at::empty_symint(bias->sym_sizes(), bias->options());
  return wanted({dh, dw, db});
}
at::Tensor ffn_infer_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t) {
  return at::empty_symint(x.sym_sizes(), x.options());
}
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> ffn_train_meta(const at::Tensor& x, const at::Tensor& wg,
                                                                          const at::Tensor&, const at::Tensor&, int64_t) {
  const std::vector<c10::SymInt> inner{x.sym_size(0), sym8(wg.sym_size(0))};
  auto mid = [&] { return at::empty_symint(inner, x.options()); };
  return {at::empty_symint(x.sym_sizes(), x.options()), mid(), mid(), mid()};
}
std::vector<at::Tensor> ffn_backward_meta(const at::Tensor&, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu,
                                          const at::Tensor& wd, const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t,
                                          bool need_x, bool need_g, bool need_u, bool need_d) {
  auto like = [&](bool need, const at::Tensor& t) { return need ? at::empty_symint(t.sym_sizes(), x.options()) : at::Tensor(); };
  return wanted({like(need_x, x), like(need_g, wg), like(need_u, wu), like(need_d, wd)});
}

// The operators that have kernels, reached through the dispatcher, so that tracing sees them.
template <class F>
c10::TypedOperatorHandle<F> op_of(const char* name, F*) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
const auto& lce_forward_op() {
  static const auto op = op_of("mihvd::_linear_cross_entropy", &lce_forward);
  return op;
}
const auto& lce_backward_op() {
  static const auto op = op_of("mihvd::_linear_cross_entropy_backward", &lce_backward);
  return op;
}
const auto& ffn_infer_op() {
  static const auto op = op_of("mihvd::_gated_ffn", &ffn_infer);
  return op;
}
const auto& ffn_train_op() {
  static const auto op = op_of("mihvd::_gated_ffn_train", &ffn_train);
  return op;
}
const auto& ffn_backward_op() {
  static const auto op = op_of("mihvd::_gated_ffn_backward", &ffn_backward);
  return op;
}

// ------------------------------------------------------------------------------------------ //
// Autograd. In C++, since a small call's time is the host's. A gradient that is itself to be differentiated
// goes through Once, whose backward refuses.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Once : torch::autograd::Function<Once> {
  static at::Tensor forward(AutogradContext*, const at::Tensor& grad, const at::Tensor&) { return grad.view_as(grad); }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "linear_cross_entropy / gated_ffn: their gradients cannot be differentiated again");
    return {};
  }
};
void once(const at::Tensor& gout, variable_list& grads) {
  if (!at::GradMode::is_enabled()) return;
  const at::Tensor any = gout.detach().requires_grad_(true);
  for (at::Tensor& t : grads)
    if (t.defined()) t = Once::apply(t, any);
}

// A forward-mode derivative has no formula here, and would be taken for zero wherever a call passes the
// autograd function by.
void refuse_tangents(const char* op, std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), op, ": forward-mode derivatives are not implemented");
}

// Called by a backward pass before anything else runs. While a stream is captured, the engine would make a
// leaf's gradient accumulator that an eager graph on the default stream still holds wait there for the
// captured stream, which invalidates the capture inside the engine and ends the process: refused
// here, with the graph behind this node searched for such leaves.
void refuse_eager_leaves(const char* op) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  C10_HIP_CHECK(hipStreamIsCapturing(cur_stream(), &status));
  if (status == hipStreamCaptureStatusNone) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  std::vector<torch::autograd::Node*> stack{node.get()};
  std::unordered_set<torch::autograd::Node*> seen;
  while (!stack.empty()) {
    torch::autograd::Node* n = stack.back();
    stack.pop_back();
    if (!seen.insert(n).second) continue;
    if (auto* acc = dynamic_cast<torch::autograd::AccumulateGrad*>(n)) {
      const auto stream = acc->stream();
      if (acc->variable.is_cuda())
        TORCH_CHECK(stream && stream->id() != c10::hip::getDefaultHIPStream(acc->variable.get_device()).id(), op,
                    ": the backward pass is being captured while an eager autograd graph of the same leaves is alive on "
                    "the default stream; drop that graph (its loss and outputs), or run it on a side stream");
      continue;
    }
    for (const auto& e : n->next_edges())
      if (e.function) stack.push_back(e.function.get());
  }
}

// The wanted gradients back in their places.
template <size_t N>
variable_list spread(std::vector<at::Tensor> got, const bool (&need)[N]) {
  variable_list r(N);
  size_t k = 0;
  for (size_t i = 0; i < N; ++i)
    if (need[i]) r[i] = std::move(got[k++]);
  return r;
}

struct LceFunction : torch::autograd::Function<LceFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& h, const at::Tensor& w, const at::Tensor& labels,
                            const c10::optional<at::Tensor>& bias, int64_t ignore_index, int64_t reduction) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [loss, hc, meta, lse] = lce_forward_op().call(h, w, labels, bias, ignore_index, reduction);
    ctx->save_for_backward({hc, w, meta, lse, bias ? *bias : at::Tensor()});
    ctx->saved_data["reduction"] = reduction;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list gout) {
    refuse_eager_leaves("linear_cross_entropy");
    const variable_list t = ctx->get_saved_variables();
    c10::optional<at::Tensor> bias;
    if (t[4].defined()) bias = t[4];
    const bool need[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), bias && ctx->needs_input_grad(3)};
    variable_list grads;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      grads = spread(lce_backward_op().call(gout[0], t[0], t[1], bias, t[2], t[3], ctx->saved_data["reduction"].toInt(), need[0],
                                            need[1], need[2]),
                     need);
    }
    once(gout[0], grads);
    return {grads[0], grads[1], at::Tensor(), grads[2], at::Tensor(), at::Tensor()};
  }
};

at::Tensor linear_cross_entropy(const at::Tensor& h, const at::Tensor& w, const at::Tensor& labels,
                                const c10::optional<at::Tensor>& bias, int64_t ignore_index, int64_t reduction) {
  refuse_tangents("linear_cross_entropy", {&h, &w, bias ? &*bias : &w});
  if (at::GradMode::is_enabled() && (h.requires_grad() || w.requires_grad() || (bias && bias->requires_grad())))
    return LceFunction::apply(h, w, labels, bias, ignore_index, reduction);
  at::AutoDispatchBelowADInplaceOrView below;
  return std::get<0>(lce_forward_op().call(h, w, labels, bias, ignore_index, reduction));
}

struct FfnFunction : torch::autograd::Function<FfnFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu,
                            const at::Tensor& wd, int64_t act) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, g, u, h] = ffn_train_op().call(x, wg, wu, wd, act);
    ctx->save_for_backward({x, wg, wu, wd, g, u, h});
    ctx->saved_data["act"] = act;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    refuse_eager_leaves("gated_ffn");
    const variable_list t = ctx->get_saved_variables();
    const bool need[4] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2), ctx->needs_input_grad(3)};
    variable_list grads;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      grads = spread(ffn_backward_op().call(dy[0], t[0], t[1], t[2], t[3], t[4], t[5], t[6], ctx->saved_data["act"].toInt(),
                                            need[0], need[1], need[2], need[3]),
                     need);
    }
    once(dy[0], grads);
    grads.emplace_back();
    return grads;
  }
};

at::Tensor gated_ffn(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t act) {
  refuse_tangents("gated_ffn", {&x, &wg, &wu, &wd});
  if (at::GradMode::is_enabled() && (x.requires_grad() || wg.requires_grad() || wu.requires_grad() || wd.requires_grad()))
    return FfnFunction::apply(x, wg, wu, wd, act);
  at::AutoDispatchBelowADInplaceOrView below;
  return ffn_infer_op().call(x, wg, wu, wd, act);
}

// ------------------------------------------------------------------------------------------ //
// Newton-Schulz

constexpr int64_t NS_ELEMS = int64_t(1) << 28;  // elements of X per launch group (bounds the workspace)

inline int64_t up64(int64_t x) { return cdiv(x, 64) * 64; }

// Adds a matrix to the group, unless it is full.
bool ns_add(NsGroup& g, int64_t rows, int64_t cols, const void* src, void* dst, float* mom, float step) {
  const int64_t len = up64(std::max(rows, cols)), side = up64(std::min(rows, cols));
  const int64_t off = g.count ? g.m[g.count - 1].off + (int64_t)g.planes * g.side * g.m[g.count - 1].len : 0;
  if (g.count && (g.count == NS_MAX || g.side != side || off / g.planes + side * len > NS_ELEMS)) return false;
  g.side = (int)side;
  g.m[g.count++] = NsMat{src, dst, mom, (int)rows, (int)cols, (int)len, off, step};
  return true;
}

void ns_launch(NsGroup& g, const NsParams& p, const at::TensorOptions& opt) {
  if (!g.count) return;
  const NsMat& last = g.m[g.count - 1];
  const int64_t all = last.off + (int64_t)g.planes * g.side * last.len;
  const int64_t sq = (int64_t)g.count * g.planes * g.side * g.side;
  const auto h = opt.dtype(at::kHalf);
  at::Tensor x0 = at::empty({all}, h), x1, gram, poly;
  if (p.steps > 0) {
    gram = at::empty({sq}, h);
    poly = at::empty({sq}, h);
  }
  if (p.steps > 1) x1 = at::empty({all}, h);
  at::Tensor part = at::empty({g.count * NS_PART}, opt.dtype(at::kDouble));
  ns_run(g, p, NsScratch{m16(x0), m16(x1), m16(gram), m16(poly), part.data_ptr<double>()}, cur_stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
  g.count = 0;
}

void ns_check_sides(int64_t rows, int64_t cols) {
  TORCH_CHECK_VALUE(rows <= MAX_LD && cols <= MAX_LD, "orthogonalize: sides above ", MAX_LD, " are not supported");
}

at::Tensor newton_schulz(const at::Tensor& x_in, int64_t steps, double a, double b, double c, double eps, bool split) {
  TORCH_CHECK_VALUE(x_in.dim() == 3 && x_in.is_cuda(), "newton_schulz: a [batch, rows, cols] GPU tensor is expected");
  const auto ty = x_in.scalar_type();
  TORCH_CHECK_TYPE(ty == at::kFloat || ty == at::kBFloat16 || ty == at::kHalf,
                   "newton_schulz: float32, bfloat16 or float16 expected (got ", ty, ")");
  TORCH_CHECK_VALUE(steps >= 0 && steps <= 100, "newton_schulz: steps must be within 0..100");
  c10::DeviceGuard guard(x_in.device());
  at::Tensor x = x_in.contiguous(), out = at::empty_like(x);
  if (x.numel() == 0) return out;
  NsParams p{};
  p.steps = (int)steps;
  p.a = (float)a, p.b = (float)b, p.c = (float)c, p.eps = (float)eps;
  p.src_kind = ty == at::kFloat ? 0 : ty == at::kBFloat16 ? 1 : 2;
  const int64_t B = x.size(0), bytes = x.size(1) * x.size(2) * x.element_size();
  ns_check_sides(x.size(1), x.size(2));
  NsGroup g{};
  g.planes = split ? 2 : 1;
  for (int64_t i = 0; i < B; ++i) {
    auto add = [&] {
      return ns_add(g, x.size(1), x.size(2), static_cast<const char*>(x.data_ptr()) + i * bytes,
                    static_cast<char*>(out.data_ptr()) + i * bytes, nullptr, 0.f);
    };
    if (!add()) {
      ns_launch(g, p, x.options());
      add();
    }
  }
  ns_launch(g, p, x.options());
  return out;
}

// scale_mode: 0 sqrt(max(1, rows / cols)), 1 0.2 sqrt(max(rows, cols))
void muon_step(std::vector<at::Tensor> ps, std::vector<at::Tensor> gs, std::vector<at::Tensor> ms, double lr,
               double momentum, bool nesterov, double weight_decay, int64_t steps, double a, double b, double c, double eps,
               int64_t scale_mode, bool split) {
  TORCH_CHECK_VALUE(ps.size() == gs.size() && ps.size() == ms.size(), "muon_step: list lengths");
  TORCH_CHECK_VALUE(steps >= 0 && steps <= 100, "muon_step: steps must be within 0..100");
  // matrices whose smaller sides agree (padded) run together
  std::map<std::tuple<int, int64_t>, std::vector<size_t>> groups;
  for (size_t i = 0; i < ps.size(); ++i) {
    TORCH_CHECK_VALUE(ps[i].dim() >= 2, "muon_step: parameters must be matrices");
    for (const at::Tensor* t : {&ps[i], &gs[i], &ms[i]})
      TORCH_CHECK_VALUE(t->is_cuda() && t->scalar_type() == at::kFloat && t->is_contiguous() &&
                            t->sizes() == ps[i].sizes() && t->device() == ps[i].device(),
                        "muon_step: contiguous fp32 GPU tensors of equal shapes expected");
    if (ps[i].numel() == 0) continue;
    const int64_t rows = ps[i].size(0), cols = ps[i].numel() / rows;
    ns_check_sides(rows, cols);
    groups[{(int)ps[i].get_device(), up64(std::min(rows, cols))}].push_back(i);
  }
  NsParams p{};
  p.steps = (int)steps;
  p.a = (float)a, p.b = (float)b, p.c = (float)c, p.eps = (float)eps;
  p.muon = 1;
  p.momentum = (float)momentum, p.decay = (float)(1.0 - lr * weight_decay);
  p.nesterov = nesterov;
  for (const auto& kv : groups) {
    const at::TensorOptions opt = ps[kv.second[0]].options();
    c10::DeviceGuard guard(opt.device());
    NsGroup g{};
    g.planes = split ? 2 : 1;
    for (const size_t k : kv.second) {
      const int64_t rows = ps[k].size(0), cols = ps[k].numel() / rows;
      const double s = scale_mode == 0 ? std::sqrt(std::max(1.0, (double)rows / (double)cols))
                                       : 0.2 * std::sqrt((double)std::max(rows, cols));
      auto add = [&] {
        return ns_add(g, rows, cols, gs[k].data_ptr<float>(), ps[k].data_ptr<float>(), ms[k].data_ptr<float>(),
                      (float)(lr * s));
      };
      if (!add()) {
        ns_launch(g, p, opt);
        add();
      }
    }
    ns_launch(g, p, opt);
  }
}

at::Tensor newton_schulz_meta(const at::Tensor& x, int64_t, double, double, double, double, bool) {
  return at::empty_symint(x.sym_sizes(), x.options());
}
void muon_step_meta(std::vector<at::Tensor>, std::vector<at::Tensor>, std::vector<at::Tensor>, double, double, bool, double, int64_t,
                    double, double, double, double, int64_t, bool) {}

// The weights and momenta count as changed in place: a backward pass that saved a weight before the step raises.
void muon_step_in_place(std::vector<at::Tensor> ps, std::vector<at::Tensor> gs, std::vector<at::Tensor> ms, double lr,
                        double momentum, bool nesterov, double weight_decay, int64_t steps, double a, double b, double c,
                        double eps, int64_t scale_mode, bool split) {
  {
    at::AutoDispatchBelowADInplaceOrView below;
    muon_step(ps, std::move(gs), ms, lr, momentum, nesterov, weight_decay, steps, a, b, c, eps, scale_mode, split);
  }
  for (const auto* list : {&ps, &ms})
    for (const at::Tensor& t : *list) torch::autograd::impl::bump_version(t);
}

// How a call of these sizes runs, for tests that have to reach every kernel and for reading profiles:
//   linear_cross_entropy [rows, hidden, vocabulary, bias]: tiles of the logits, dz, dh, dW; dh's splits at most; pieces
//   gated_ffn [rows, hidden, inner]: the gate product's tile (0: few rows); tile, splits of y, dWd, dWg and dWu, dx
//   orthogonalize [batch, rows, cols, planes]: tiles of X X^T, the polynomial, X's update, the last update
std::vector<int64_t> transformer_plan(c10::string_view op, std::vector<int64_t> z) {
  for (size_t i = 0; i < z.size(); ++i)
    TORCH_CHECK_VALUE(z[i] >= (op == "linear_cross_entropy" && i == 3 ? 0 : 1) && z[i] <= MAX_LD, "transformer_plan: sizes within 1..",
                      MAX_LD);
  if (op == "linear_cross_entropy" && z.size() == 4) {
    LceShape s{(int)z[0], (int)z[1], (int)up8(z[1]), (int)z[2], 0, 0, 0};
    LceScratch x{};
    lce_plan(s);
    lce_pieces(s, x);
    lce_plan_backward(s, x, z[3] != 0);
    return {s.tile, x.dz_tile, x.dh_tile, x.dw_tile, x.splits, cdiv(s.V, x.piece)};
  }
  if (op == "gated_ffn" && z.size() == 3) {
    const FfnPlan p = ffn_plan({(int)z[0], (int)z[1], (int)up8(z[1]), (int)z[2], (int)up8(z[2])});
    std::vector<int64_t> r{p.gate};
    for (int i = 0; i < 4; ++i) r.insert(r.end(), {p.tile[i], p.splits[i]});
    return r;
  }
  TORCH_CHECK_VALUE(op == "orthogonalize" && z.size() == 4 && z[0] <= NS_MAX && z[3] <= 2,
                    "transformer_plan: linear_cross_entropy, gated_ffn or orthogonalize and its sizes");
  NsGroup g{};
  g.planes = (int)z[3];
  for (int64_t i = 0; i < z[0]; ++i) ns_add(g, z[1], z[2], nullptr, nullptr, nullptr, 0.f);
  const NsPlan p = ns_plan(g);
  return {p.gram, p.poly, p.update, p.last};
}

}  // namespace
}  // namespace mihvd

TORCH_LIBRARY_FRAGMENT(mihvd, m) {
  m.def("transformer_plan(str op, int[] sizes) -> int[]", &mihvd::transformer_plan);
  m.def("linear_cross_entropy(Tensor hidden, Tensor weight, Tensor labels, Tensor? bias, int ignore_index, int reduction) "
        "-> Tensor", &mihvd::linear_cross_entropy);
  m.def("gated_ffn(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, int act) -> Tensor", &mihvd::gated_ffn);
  // what those two are made of: loss, packed rows, row numbers and labels, (maximum, log of the sum); y, g, u, h
  m.def("_linear_cross_entropy(Tensor hidden, Tensor weight, Tensor labels, Tensor? bias, int ignore_index, int reduction) "
        "-> (Tensor, Tensor, Tensor, Tensor)");
  m.def("_linear_cross_entropy_backward(Tensor grad, Tensor rows, Tensor weight, Tensor? bias, Tensor meta, Tensor lse, "
        "int reduction, bool need_hidden, bool need_weight, bool need_bias) -> Tensor[]");
  m.def("_gated_ffn(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, int act) -> Tensor");
  m.def("_gated_ffn_train(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, int act) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("_gated_ffn_backward(Tensor grad, Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, Tensor g, Tensor u, Tensor h, "
        "int act, bool need_x, bool need_gate, bool need_up, bool need_down) -> Tensor[]");
  m.def("newton_schulz(Tensor x, int steps, float a, float b, float c, float eps, bool split) -> Tensor");
  m.def("muon_step(Tensor(a!)[] p, Tensor[] g, Tensor(b!)[] m, float lr, float momentum, bool nesterov, "
        "float weight_decay, int steps, float a, float b, float c, float eps, int scale_mode, bool split) -> ()");
}

TORCH_LIBRARY_IMPL(mihvd, CUDA, m) {
  m.impl("_linear_cross_entropy", &mihvd::lce_forward);
  m.impl("_linear_cross_entropy_backward", &mihvd::lce_backward);
  m.impl("_gated_ffn", &mihvd::ffn_infer);
  m.impl("_gated_ffn_train", &mihvd::ffn_train);
  m.impl("_gated_ffn_backward", &mihvd::ffn_backward);
  m.impl("newton_schulz", &mihvd::newton_schulz);
  m.impl("muon_step", &mihvd::muon_step);
}

TORCH_LIBRARY_IMPL(mihvd, Meta, m) {
  m.impl("_linear_cross_entropy", &mihvd::lce_forward_meta);
  m.impl("_linear_cross_entropy_backward", &mihvd::lce_backward_meta);
  m.impl("_gated_ffn", &mihvd::ffn_infer_meta);
  m.impl("_gated_ffn_train", &mihvd::ffn_train_meta);
  m.impl("_gated_ffn_backward", &mihvd::ffn_backward_meta);
  m.impl("newton_schulz", &mihvd::newton_schulz_meta);
  m.impl("muon_step", &mihvd::muon_step_meta);
}

TORCH_LIBRARY_IMPL(mihvd, ADInplaceOrView, m) { m.impl("muon_step", &mihvd::muon_step_in_place); }
