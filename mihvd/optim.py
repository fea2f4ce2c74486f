"""Optimizers with the reference's exact update rules.

``TFAdam`` implements ``tf.train.AdamOptimizer`` (horovod/tensorflow_mnist.py:130), which differs
from ``torch.optim.Adam`` in where epsilon sits:

    lr_t = lr * sqrt(1 - beta2^t) / (1 - beta1^t)
    m    = beta1 * m + (1 - beta1) * g
    v    = beta2 * v + (1 - beta2) * g^2
    p   -= lr_t * m / (sqrt(v) + epsilon)          # epsilon = 1e-8 ("epsilon hat")

(Keras ``Adam`` — tensorflow_mnist_gpu.py:134 — is the same rule with epsilon 1e-7.) The state
names match torch's Adam (``exp_avg``, ``exp_avg_sq``, ``step``) so checkpoint mapping and
``broadcast_optimizer_state`` work unchanged. The fused HIP kernel ``mihvd::adam_step`` uses the
identical rule on the flat parameter buffer.
"""
from __future__ import annotations

import functools
import math

import torch


def _fused_ok(tensors) -> bool:
    """The multi-tensor HIP kernels apply: every tensor is a contiguous fp32 GPU tensor."""
    if not tensors or not all(t.is_cuda and t.dtype == torch.float32 and t.is_contiguous() for t in tensors):
        return False
    from . import _native

    return _native.load_kernels()


def _dense(t: torch.Tensor) -> bool:
    if t.is_contiguous():
        return True
    if t.dim() == 4:
        return t.is_contiguous(memory_format=torch.channels_last)
    if t.dim() == 5:
        return t.is_contiguous(memory_format=torch.channels_last_3d)
    return False


def _flat(t: torch.Tensor) -> torch.Tensor:
    return t.as_strided((t.numel(),), (1,), t.storage_offset())


def _split_fused(*lists):
    """Partition parallel tensor lists (p, g, state...) into the ones the multi-tensor kernels can
    update — fp32 GPU tensors that are dense with identical strides (e.g. channels_last conv
    weights whose grads and slots share the layout), passed as flat views — and the indices left
    to the torch path."""
    from . import _native

    n = len(lists[0])
    ok_kernels = n > 0 and lists[0][0].is_cuda and _native.load_kernels()
    fused = [[] for _ in lists]
    rest = []
    for i in range(n):
        ts = [lst[i] for lst in lists]
        good = ok_kernels and all(
            t.is_cuda and t.dtype == torch.float32 and t.stride() == ts[0].stride() and t.shape == ts[0].shape
            and _dense(t) for t in ts)
        if good:
            for f, t in zip(fused, ts):
                f.append(_flat(t))
        else:
            rest.append(i)
    return fused, rest


class TFAdam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8):
        if lr < 0:
            raise ValueError("invalid learning rate")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            b1, b2 = group["betas"]
            params, grads, ms, vs = [], [], [], []
            step_t = None
            for p in group["params"]:
                if p.grad is None:
                    continue
                st = self.state[p]
                if not st:
                    st["step"] = torch.tensor(0.0)
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st["step"] += 1
                step_t = float(st["step"])
                params.append(p)
                grads.append(p.grad)
                ms.append(st["exp_avg"])
                vs.append(st["exp_avg_sq"])
            if not params:
                continue
            if _fused_ok(params + grads + ms + vs):
                # one multi-tensor HIP launch per 24 tensors (csrc/kernels/multi_tensor.hip), same rule
                torch.ops.mihvd.multi_tensor_adam(params, grads, ms, vs, None, int(step_t), group["lr"], b1, b2,
                                                  group["eps"], 0.0, False, 0, 1.0)
                continue
            lr_t = group["lr"] * math.sqrt(1 - b2 ** step_t) / (1 - b1 ** step_t)
            torch._foreach_mul_(ms, b1)
            torch._foreach_add_(ms, grads, alpha=1 - b1)
            torch._foreach_mul_(vs, b2)
            torch._foreach_addcmul_(vs, grads, grads, value=1 - b2)
            denom = torch._foreach_sqrt(vs)
            torch._foreach_add_(denom, group["eps"])
            torch._foreach_addcdiv_(params, ms, denom, value=-lr_t)
        return loss


class FusedAdam(torch.optim.Optimizer):
    """Adam / AdamW over arbitrary parameter lists with the multi-tensor HIP kernel.

    ``rule="torch"`` is torch.optim.Adam's update, ``rule="tf"`` the TF1 rule of ``TFAdam``;
    ``adamw=True`` decouples the weight decay. The step count of each parameter group lives in a
    device int64 tensor advanced by a tiny kernel, so ``step()`` issues no host synchronisation and
    can be captured in a HIP graph (``mihvd.graphs.CapturedStep``). Checkpoints carry the count as
    ``param_groups[i]["step"]``. Falls back to torch ops for CPU tensors.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, adamw=False, rule="torch"):
        if rule not in ("torch", "tf"):
            raise ValueError("rule must be 'torch' or 'tf'")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, adamw=adamw, rule=rule,
                                      step=0))
        self._dev_steps: dict[int, torch.Tensor] = {}

    def _group_step(self, gi, group, device):
        t = self._dev_steps.get(gi)
        if t is None or t.device != device:
            t = torch.full((1,), int(group.get("step", 0)), dtype=torch.int64, device=device)
            self._dev_steps[gi] = t
        return t

    def state_dict(self):
        for gi, group in enumerate(self.param_groups):
            if gi in self._dev_steps:
                group["step"] = int(self._dev_steps[gi].item())
        return super().state_dict()

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        for gi, group in enumerate(self.param_groups):
            if gi in self._dev_steps:
                self._dev_steps[gi].fill_(int(group.get("step", 0)))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for gi, group in enumerate(self.param_groups):
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            for p in params:
                st = self.state[p]
                if not st:
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            grads = [p.grad for p in params]
            ms = [self.state[p]["exp_avg"] for p in params]
            vs = [self.state[p]["exp_avg_sq"] for p in params]
            b1, b2 = group["betas"]
            rule = 0 if group["rule"] == "tf" else 1
            from . import _native

            if params[0].is_cuda and _native.load_kernels():
                stp = self._group_step(gi, group, params[0].device)
                torch.ops.mihvd.bump_step_(stp)
                (fp, fg, fm, fv), idx = _split_fused(params, grads, ms, vs)
                if fp:
                    torch.ops.mihvd.multi_tensor_adam(fp, fg, fm, fv, stp, 0, group["lr"], b1, b2, group["eps"],
                                                      group["weight_decay"], bool(group["adamw"]), rule, 1.0)
                if not idx:
                    continue
                t = int(stp.item())  # tensors the kernel cannot take: torch path (one host read)
            else:
                group["step"] = int(group.get("step", 0)) + 1
                t = group["step"]
                idx = range(len(params))
            bc1, bc2 = 1 - b1 ** t, 1 - b2 ** t
            for i in idx:
                p, g, m, v = params[i], grads[i], ms[i], vs[i]
                if group["weight_decay"]:
                    if group["adamw"]:
                        p.mul_(1 - group["lr"] * group["weight_decay"])
                    else:
                        g = g.add(p, alpha=group["weight_decay"])
                m.mul_(b1).add_(g, alpha=1 - b1)
                v.mul_(b2).addcmul_(g, g, value=1 - b2)
                if rule == 0:
                    p.addcdiv_(m, v.sqrt().add_(group["eps"]), value=-group["lr"] * math.sqrt(bc2) / bc1)
                else:
                    p.addcdiv_(m, (v / bc2).sqrt().add_(group["eps"]), value=-group["lr"] / bc1)
        return loss


class FusedSGD(torch.optim.Optimizer):
    """SGD with momentum / dampening / Nesterov / weight decay (torch.optim.SGD semantics) with the
    multi-tensor HIP kernel; no host synchronisation after the first step (capturable)."""

    def __init__(self, params, lr=0.1, momentum=0.0, dampening=0.0, weight_decay=0.0, nesterov=False):
        super().__init__(params, dict(lr=lr, momentum=momentum, dampening=dampening, weight_decay=weight_decay,
                                      nesterov=nesterov))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            mom = group["momentum"]
            first = False
            bufs = []
            if mom:
                for p in params:
                    st = self.state[p]
                    if "momentum_buffer" not in st:
                        st["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                        first = True  # the group's buffers are created together, on its first step
                    bufs.append(st["momentum_buffer"])
            grads = [p.grad for p in params]
            if mom:
                (fp, fg, fb), idx = _split_fused(params, grads, bufs)
            else:
                (fp, fg), idx = _split_fused(params, grads)
                fb = []
            if fp:
                torch.ops.mihvd.multi_tensor_sgd(fp, fg, fb, group["lr"], mom, group["dampening"],
                                                 group["weight_decay"], bool(group["nesterov"]), first, 1.0)
            for i in idx:
                p, g = params[i], grads[i]
                d = g.add(p, alpha=group["weight_decay"]) if group["weight_decay"] else g
                if mom:
                    b = bufs[i]
                    if first:
                        b.copy_(d)
                    else:
                        b.mul_(mom).add_(d, alpha=1 - group["dampening"])
                    d = d.add(b, alpha=mom) if group["nesterov"] else b
                p.add_(d, alpha=-group["lr"])
        return loss


# Published with the update rule (K. Jordan et al., "Muon: an optimizer for hidden layers in neural networks", 2024), as
# is the scale sqrt(max(1, rows / cols)); 0.2 sqrt(max(rows, cols)) is from J. Liu et al., "Muon is scalable for
# LLM training", 2025.
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _ns_coefficients(op, coefficients):
    """The three as floats."""
    if len(coefficients) != 3:
        raise ValueError("%s: three coefficients are needed" % op)
    abc = tuple(float(v) for v in coefficients)
    if not sum(map(abs, abc)) <= 15:
        raise ValueError("%s: the coefficients' magnitudes must not add up to more than 15 (got %s)" % (op, abc))
    return abc


@functools.lru_cache(maxsize=64)
def _ns_reach(steps, a, b, c):
    """The largest value that any of the matrices X, A = X X^T and a I + b A + c A A can hold before the last
    step is done: their elements lie below their largest eigenvalues, and X's singular values start within one.
    A step takes a singular value s to s q(s^2), q(t) = a + b t + c t^2; each maximum over [0, top] is at an
    end or where the derivative vanishes."""

    def most(f, top, roots):
        return max(abs(f(t)) for t in (0.0, top, *[t for t in roots if 0.0 < t < top]))

    def q(t):
        return a + t * (b + t * c)

    disc = 9 * b * b - 20 * a * c  # (s q(s^2))' = a + 3 b t + 5 c t^2
    if c:
        turns = [(-3 * b + sign * math.sqrt(disc)) / (10 * c) for sign in (1, -1)] if disc >= 0 else []
        vertex = [-b / (2 * c)]
    else:
        turns, vertex = [-a / (3 * b)] if b else [], []
    top, reach = 1.0, 1.0
    for k in range(steps):
        reach = max(reach, top, top * top, most(q, top * top, vertex))
        if reach > 1e9:
            break
        top = most(lambda t: math.sqrt(t) * q(t), top * top, turns)
    return reach


def _ns_check_range(op, steps, coefficients):
    """The kernels hold those matrices in fp16 scaled by 2^12, which ends at 16."""
    reach = _ns_reach(steps, *coefficients)
    if not reach <= 15:
        raise ValueError("%s: %d steps with the coefficients %s can reach values of %.3g; the GPU's fp16 planes hold them "
                         "up to 15" % (op, steps, tuple(coefficients), reach))


def orthogonalize(x: torch.Tensor, steps: int = 5, coefficients=NS_COEFFICIENTS, eps: float = 1e-7,
                  precision: str | None = None) -> torch.Tensor:
    """The matrix (or each matrix of a batch, [..., rows, cols]) with its singular values driven towards
    one by ``steps`` Newton-Schulz steps:

        X = x / (|x|_F + eps);   A = X X^T;   X <- a X + (b A + c A A) X        (a, b, c = coefficients)

    (on the smaller side; the default coefficients leave the singular values near 1 within about 0.3).
    The result has ``x``'s type and shape, and takes no part in autograd (``x`` is detached). ``precision``:
    ``"fp16"`` — one fp16 product with fp32 accumulation per step, the default for 16-bit inputs, off by about
    0.0016 of the result's norm — or ``"fp32"`` — three products over split values (22 bits), the default for
    fp32. On the GPU it runs csrc/kernels/newton_schulz.hip, and coefficients whose steps can pass what fp16
    planes hold of X, A and the polynomial are refused; CPU tensors take the formula in fp32 torch operations.
    """
    if x.dim() < 2:
        raise ValueError("orthogonalize: a matrix or a batch of matrices is needed (got shape %s)" % (tuple(x.shape),))
    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError("orthogonalize: float32, bfloat16 or float16 is needed (got %s)" % x.dtype)
    if precision not in (None, "fp32", "fp16"):
        raise ValueError("orthogonalize: precision must be 'fp32' or 'fp16' (got %r)" % (precision,))
    if not 0 <= int(steps) <= 100:
        raise ValueError("orthogonalize: steps must be within 0..100 (got %r)" % (steps,))
    a, b, c = _ns_coefficients("orthogonalize", coefficients)
    if not x.numel():
        return x.detach().clone()
    if x.is_cuda:
        from . import _native

        _ns_check_range("orthogonalize", int(steps), (a, b, c))
        _native.require_kernels()
        split = precision == "fp32" or (precision is None and x.dtype == torch.float32)
        out = torch.ops.mihvd.newton_schulz(x.detach().reshape(-1, *x.shape[-2:]), int(steps), a, b, c, float(eps), split)
        return out.view(x.shape)
    z = x.detach().double()  # the norm's squares may leave fp32's range
    z = (z / (torch.linalg.vector_norm(z, dim=(-2, -1), keepdim=True) + eps)).float()
    tall = z.shape[-2] > z.shape[-1]
    if tall:
        z = z.transpose(-2, -1)
    for _ in range(int(steps)):
        gram = z @ z.transpose(-2, -1)
        z = a * z + (b * gram + c * (gram @ gram)) @ z
    return (z.transpose(-2, -1) if tall else z).to(x.dtype).contiguous()


class Muon(torch.optim.Optimizer):
    """Momentum whose update is orthogonalised (:func:`orthogonalize`), for the matrices of a model:

        m = momentum * m + g;   u = g + momentum * m  (``nesterov``)  or  m
        p = p (1 - lr * weight_decay) - lr * s * orthogonalize(u)

    ``scale="spectral"``: s = sqrt(max(1, rows / cols)); ``"rms"``: s = 0.2 sqrt(max(rows, cols)), which
    gives updates of AdamW's size, so that its learning rate and decay carry over. Parameters of more
    than two dimensions count as [first, rest]. Vectors, embeddings and heads belong to another
    optimizer (``FusedAdam``); parameters of fewer than two dimensions are refused.

    fp32 contiguous GPU parameters take one fused path (``torch.ops.mihvd.muon_step``: matrices of like
    smaller sides run together, momentum, products and weight update in the kernels, no host
    synchronisation, capturable from the second step on, with the learning rate it then has); others use
    torch operations around :func:`orthogonalize`. The momentum is fp32 for parameters of any type (a sum over
    many steps loses in 16 bits what is small beside it), and so is the update; a 16-bit parameter is
    rounded once a step. ``precision`` is that of the products (see there).
    """

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, ns_steps=5,
                 ns_coefficients=NS_COEFFICIENTS, eps=1e-7, scale="spectral", precision="fp32"):
        super().__init__(params, self._checked(dict(
            lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, ns_steps=ns_steps,
            ns_coefficients=ns_coefficients, eps=eps, scale=scale, precision=precision)))

    @staticmethod
    def _checked(group):
        """A group's options (the constructor's or its own), checked."""
        if group["lr"] < 0 or group["weight_decay"] < 0 or not 0 <= group["momentum"] < 1:
            raise ValueError("Muon: lr and weight_decay must not be negative, momentum must be within [0, 1)")
        if not 0 <= int(group["ns_steps"]) <= 100:
            raise ValueError("Muon: ns_steps must be within 0..100")
        if group["scale"] not in ("spectral", "rms"):
            raise ValueError("Muon: scale must be 'spectral' or 'rms'")
        if group["precision"] not in ("fp32", "fp16"):
            raise ValueError("Muon: precision must be 'fp32' or 'fp16'")
        group["ns_steps"] = int(group["ns_steps"])
        group["ns_coefficients"] = _ns_coefficients("Muon", group["ns_coefficients"])
        return group

    def add_param_group(self, group):
        super().add_param_group(group)
        try:
            params = self._checked(self.param_groups[-1])["params"]
            if len({id(p) for p in params}) != len(params):
                raise ValueError("Muon: a parameter is listed twice (matrices run together: both updates would run at once)")
            for p in params:
                if p.dim() < 2:
                    raise ValueError("Muon: parameters must have at least two dimensions (got shape %s); give vectors to "
                                     "another optimizer" % (tuple(p.shape),))
                if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
                    raise TypeError("Muon: parameters must be float32, bfloat16 or float16 (got %s)" % p.dtype)
        except (TypeError, ValueError):
            self.param_groups.pop()
            raise

    def load_state_dict(self, state_dict):
        for group in state_dict["param_groups"]:
            self._checked(dict(self.defaults, **group))
        super().load_state_dict(state_dict)
        # torch has cast the state to its parameters' types: the momenta of 16-bit ones come back in fp32
        loaded = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i, p in zip(loaded, [p for group in self.param_groups for p in group["params"]]):
            m = state_dict["state"].get(i, {}).get("momentum_buffer")
            if m is not None and p.dtype != torch.float32:
                self.state[p]["momentum_buffer"] = m.to(device=p.device, dtype=torch.float32)

    @torch.no_grad()
    def step(self, closure=None):
        for group in self.param_groups:  # before anything is written
            self._checked(group)
            if any(p.is_cuda for p in group["params"]):
                _ns_check_range("Muon", group["ns_steps"], group["ns_coefficients"])
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            fused = ([], [], [])
            for p in params:
                st = self.state[p]
                if "momentum_buffer" not in st:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("Muon: the first step of a parameter makes its momentum, which every replay "
                                           "would clear; run one step before capturing")
                    st["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
                m = st["momentum_buffer"]
                if p.grad.is_sparse:
                    raise RuntimeError("Muon: sparse gradients are not supported")
                if all(t.is_cuda and t.dtype == torch.float32 and t.is_contiguous() for t in (p, p.grad, m)):
                    for lst, t in zip(fused, (p, p.grad, m)):
                        lst.append(t)
                else:
                    self._plain(group, p, m)
            if fused[0]:
                from . import _native

                _native.require_kernels()
                a, b, c = group["ns_coefficients"]
                torch.ops.mihvd.muon_step(*fused, float(group["lr"]), group["momentum"], bool(group["nesterov"]),
                                          group["weight_decay"], group["ns_steps"], a, b, c, group["eps"],
                                          0 if group["scale"] == "spectral" else 1, group["precision"] == "fp32")
        return loss

    @staticmethod
    def _plain(group, p, m):
        g, mu, lr = p.grad.float(), group["momentum"], group["lr"]
        m.mul_(mu).add_(g)
        u = g.add(m, alpha=mu) if group["nesterov"] else m
        rows, cols = p.shape[0], p.numel() // max(1, p.shape[0])
        if not p.numel():
            return
        s = math.sqrt(max(1.0, rows / cols)) if group["scale"] == "spectral" else 0.2 * math.sqrt(max(rows, cols))
        o = orthogonalize(u.reshape(rows, cols), group["ns_steps"], group["ns_coefficients"], group["eps"],
                          group["precision"])
        w = p.float()  # p itself where it is fp32
        w.mul_(1.0 - lr * group["weight_decay"]).add_(o.view(p.shape), alpha=-lr * s)
        if w is not p:
            p.copy_(w)
