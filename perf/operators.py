"""Measured cases of the transformer-step operators: the vocabulary projection with its cross entropy
(``mihvd.ops.linear_cross_entropy``), the gated feed-forward block (``mihvd.ops.gated_ffn``) and the
orthogonalised update (``mihvd.optim.orthogonalize`` / ``mihvd.optim.Muon``).

Each case runs in two forms on the same inputs: the plain one (``own = False``: elementary torch
operations in 32 bits, rounded once at the end) and the framework's (``own = True``).
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_NS = (3.4445, -4.7750, 2.0315)


def listed():
    return [
        # masked-LM head of one short sequence: 15 % of 128 positions, the latency end of training
        dict(name="lce_mlm_20", op="lce", dtype="bf16", rows=20, labelled=20, hidden=768, vocab=30522, bias=True,
             train=True),
        # masked-LM head of the stress benchmark's batch (16 x 512, masked positions gathered)
        dict(name="lce_mlm_1229", op="lce", dtype="bf16", rows=1229, labelled=1229, hidden=768, vocab=30522, bias=True,
             train=True),
        # the same batch with the head on every position, 15 % of them labelled; fp16 under a loss scale
        dict(name="lce_mlm_all_fp16", op="lce", dtype="fp16", rows=8192, labelled=1229, hidden=768, vocab=30522,
             bias=True, train=True),
        # per-token losses of an evaluation pass: forward only, a ragged vocabulary
        dict(name="lce_eval_ragged", op="lce", dtype="bf16", rows=4095, labelled=4000, hidden=1000, vocab=50001,
             bias=False, train=False),
        # next-token training: every position labelled, a large vocabulary
        dict(name="lce_causal_8192", op="lce", dtype="bf16", rows=8192, labelled=8192, hidden=1024, vocab=65536,
             bias=False, train=True),
        # one token through the block, as in stepwise generation
        dict(name="ffn_serve_1", op="ffn", dtype="bf16", rows=1, hidden=768, inner=2048, act="silu", train=False),
        # the stress benchmark's batch (16 x 512) through one gated layer, with gradients
        dict(name="ffn_train_8192", op="ffn", dtype="bf16", rows=8192, hidden=768, inner=2048, act="gelu", train=True),
        # ragged sizes in fp16 under a loss scale
        dict(name="ffn_train_ragged", op="ffn", dtype="fp16", rows=1237, hidden=1000, inner=2730, act="silu",
             train=True),
        # a long batch of a wider model
        dict(name="ffn_train_16384", op="ffn", dtype="bf16", rows=16384, hidden=2048, inner=5632, act="silu",
             train=True),
        # one square projection in fp32: the smallest update, where launches count
        dict(name="orth_fp32_768", op="orth", dtype="fp32", batch=1, rows=768, cols=768),
        # the stacked attention projections of twelve layers, 16-bit
        dict(name="orth_bf16_12x2304x768", op="orth", dtype="bf16", batch=12, rows=2304, cols=768),
        # a whole optimizer step over the matrices of six gated encoder layers, fp32
        dict(name="muon_6_layers", op="muon", layers=6, hidden=768, inner=2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lce", "lce", "lce", "ffn", "ffn", "ffn", "orth", "orth", "muon"])
    if op == "lce":
        top = 8192 * 65536 * 1024
        while True:
            n, k, v = _log(rng, 1, 8192), _log(rng, 64, 1024), _log(rng, 1000, 65536)
            if rng.random() < 0.5:
                k = max(64, k // 64 * 64)
            if n * k * v <= top:
                break
        part = rng.choice([1.0, 1.0, rng.uniform(0.1, 0.95)])
        return dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), rows=n, labelled=max(1, int(n * part)), hidden=k,
                    vocab=v, bias=rng.random() < 0.5, train=rng.random() < 0.7)
    if op == "ffn":
        train = rng.random() < 0.7
        n = _log(rng, 1, 16384) if train else _log(rng, 1, 256)
        k, f = _log(rng, 64, 2048), _log(rng, 128, 5632)
        if rng.random() < 0.5:
            k, f = max(64, k // 64 * 64), max(64, f // 64 * 64)
        return dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), rows=n, hidden=k, inner=f,
                    act=rng.choice(["silu", "gelu", "gelu_tanh", "relu", "sigmoid"]), train=train)
    if op == "orth":
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), batch=rng.randint(1, 12),
                    rows=_log(rng, 16, 2304), cols=_log(rng, 16, 2304))
    return dict(op=op, layers=rng.randint(1, 6), hidden=_log(rng, 64, 768), inner=_log(rng, 128, 2048))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _lce_inputs(case, seed):
    g = _gen(seed)
    dt = _DT[case["dtype"]]
    n, k, v = case["rows"], case["hidden"], case["vocab"]
    # hidden rows as a final layer norm leaves them, pulled towards their label's row of the weight;
    # an embedding-scaled weight: logits spread over a few units, the label's a few above
    w = torch.randn(v, k, device="cuda", generator=g) * (1.5 / math.sqrt(k))
    y = torch.randint(0, v, (n,), device="cuda", generator=g)
    h = torch.randn(n, k, device="cuda", generator=g) + w[y] * torch.rand(n, 1, device="cuda", generator=g) * 2.0
    drop = torch.randperm(n, device="cuda", generator=g)[case["labelled"]:]
    y[drop] = -100
    b = torch.randn(v, device="cuda", generator=g) * 0.2 if case["bias"] else None
    scale = 16384.0 if case["dtype"] == "fp16" else 1.0  # the loss scale that fp16 gradients need
    return h.to(dt), w.to(dt), y, b, scale


def _ffn_inputs(case, seed):
    g = _gen(seed)
    dt = _DT[case["dtype"]]
    n, k, f = case["rows"], case["hidden"], case["inner"]
    x = torch.randn(n, k, device="cuda", generator=g)
    wg = torch.randn(f, k, device="cuda", generator=g) / math.sqrt(k)
    wu = torch.randn(f, k, device="cuda", generator=g) / math.sqrt(k)
    wd = torch.randn(k, f, device="cuda", generator=g) / math.sqrt(f)
    dy = torch.randn(n, k, device="cuda", generator=g) * 0.1 if case["train"] else None
    return [None if t is None else t.to(dt) for t in (x, wg, wu, wd, dy)]


def _update_like(g, *shape):
    """A gradient-like matrix: a few strong directions over a noise floor."""
    *lead, m, n = shape
    r = max(1, min(m, n) // 16)
    a = torch.randn(*lead, m, r, device="cuda", generator=g)
    b = torch.randn(*lead, r, n, device="cuda", generator=g)
    return (a @ b) / math.sqrt(r) * 1e-2 + torch.randn(*shape, device="cuda", generator=g) * 3e-3


def _orth_inputs(case, seed):
    return _update_like(_gen(seed), case["batch"], case["rows"], case["cols"]).to(_DT[case["dtype"]])


_MUON = dict(lr=0.02, momentum=0.95, weight_decay=0.01)


def _muon_shapes(case):
    h, f = case["hidden"], case["inner"]
    return [(3 * h, h), (h, h), (f, h), (f, h), (h, f)] * case["layers"]


def _muon_inputs(case, seed):
    g = _gen(seed)
    shapes = _muon_shapes(case)
    p = [torch.randn(*s, device="cuda", generator=g) * 0.02 for s in shapes]
    grad = [_update_like(g, *s) for s in shapes]
    mom = [_update_like(g, *s) * 5.0 for s in shapes]
    return p, grad, mom


def prepare(case, seed):
    op = case["op"]
    if op == "lce":
        h, w, y, b, scale = _lce_inputs(case, seed)
        st = dict(case=case, h=h, w=w, y=y, b=b, scale=torch.tensor(scale, device="cuda"))
        if own and case["train"]:
            for t in (h, w, b):
                if t is not None:
                    t.requires_grad_()
        return st
    if op == "ffn":
        x, wg, wu, wd, dy = _ffn_inputs(case, seed)
        if own and case["train"]:
            for t in (x, wg, wu, wd):
                t.requires_grad_()
        return dict(case=case, x=x, wg=wg, wu=wu, wd=wd, dy=dy)
    if op == "orth":
        return dict(case=case, x=_orth_inputs(case, seed))
    p, grad, mom = _muon_inputs(case, seed)
    st = dict(case=case, p=p, grad=grad, mom=mom)
    if own:
        from mihvd.optim import Muon

        st["p"] = [torch.nn.Parameter(t) for t in p]
        for q, d in zip(st["p"], grad):
            q.grad = d
        st["opt"] = Muon(st["p"], **_MUON)
        for q, m in zip(st["p"], mom):  # a run under way: the optimizer's momentum is loaded
            st["opt"].state[q]["momentum_buffer"] = m
    return st


def _act(name, g):
    """act(g) and act'(g)."""
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if name == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-g))
        return s, s * (1.0 - s)
    if name == "relu":
        return torch.where(g > 0, g, torch.zeros_like(g)), (g > 0).to(g.dtype)
    if name == "gelu":
        c = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * c, c + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * g * g)


def _lce_plain(st):
    case, y = st["case"], st["y"]
    h, w = st["h"].float(), st["w"].float()
    z = h @ w.t()
    if st["b"] is not None:
        z = z + st["b"]
    keep = y != -100
    safe = torch.where(keep, y, torch.zeros_like(y))
    top = z.max(dim=1, keepdim=True).values
    e = torch.exp(z - top)
    s = e.sum(dim=1, keepdim=True)
    loss = (torch.log(s) + top).squeeze(1) - z.gather(1, safe[:, None]).squeeze(1)
    loss = torch.where(keep, loss, torch.zeros_like(loss))
    if not case["train"]:
        return [loss]
    count = keep.sum()
    mean = loss.sum() / count
    dz = e.div_(s)
    dz[torch.arange(len(y), device=y.device), safe] -= 1.0
    dz *= torch.where(keep, st["scale"] / count, torch.zeros_like(loss))[:, None]
    out = [mean, (dz @ w).to(st["h"].dtype), (dz.t() @ h).to(st["w"].dtype)]
    if st["b"] is not None:
        out.append(dz.sum(dim=0))
    return out


def _lce_own(st):
    from mihvd.ops import linear_cross_entropy

    if not st["case"]["train"]:
        with torch.no_grad():
            return [linear_cross_entropy(st["h"], st["w"], st["y"], st["b"], reduction="none")]
    loss = linear_cross_entropy(st["h"], st["w"], st["y"], st["b"])
    leaves = [t for t in (st["h"], st["w"], st["b"]) if t is not None]
    return [loss.detach(), *torch.autograd.grad(loss, leaves, grad_outputs=st["scale"])]


def _ffn_plain(st):
    case = st["case"]
    dt = st["x"].dtype
    x, wg, wu, wd = (st[k].float() for k in ("x", "wg", "wu", "wd"))
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _act(case["act"], g)
    h = a * u
    y = (h @ wd.t()).to(dt)
    if not case["train"]:
        return [y]
    dy = st["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * da, dh * a
    return [y, (dg @ wg + du @ wu).to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt), (dy.t() @ h).to(dt)]


def _ffn_own(st):
    from mihvd.ops import gated_ffn

    leaves = [st[k] for k in ("x", "wg", "wu", "wd")]
    if not st["case"]["train"]:
        with torch.no_grad():
            return [gated_ffn(*leaves, activation=st["case"]["act"])]
    y = gated_ffn(*leaves, activation=st["case"]["act"])
    return [y.detach(), *torch.autograd.grad(y, leaves, grad_outputs=st["dy"])]


def _orth_plain(x):
    """Five Newton-Schulz steps on the last two dimensions, in 32 bits."""
    a, b, c = _NS
    z = x.float()
    z = z / (torch.sqrt((z * z).sum(dim=(-2, -1), keepdim=True)) + 1e-7)
    tall = z.shape[-2] > z.shape[-1]
    if tall:
        z = z.transpose(-2, -1).contiguous()
    for _ in range(5):
        gram = torch.matmul(z, z.transpose(-2, -1).contiguous())
        z = a * z + torch.matmul(b * gram + c * torch.matmul(gram, gram), z)
    return (z.transpose(-2, -1) if tall else z).contiguous()


def _muon_plain(st):
    lr, mu, wd = _MUON["lr"], _MUON["momentum"], _MUON["weight_decay"]
    for p, g, m in zip(st["p"], st["grad"], st["mom"]):
        m.mul_(mu).add_(g)
        o = _orth_plain(g + mu * m)
        p.mul_(1.0 - lr * wd).add_(o, alpha=-lr * math.sqrt(max(1.0, p.shape[0] / p.shape[1])))
    return [*st["p"], *st["mom"]]


def run(state):
    op = state["case"]["op"]
    if op == "lce":
        return _lce_own(state) if own else _lce_plain(state)
    if op == "ffn":
        return _ffn_own(state) if own else _ffn_plain(state)
    if op == "orth":
        if own:
            from mihvd.optim import orthogonalize

            return [orthogonalize(state["x"])]
        return [_orth_plain(state["x"]).to(state["x"].dtype)]
    if own:
        state["opt"].step()
        return [*(p.detach() for p in state["p"]), *state["mom"]]
    return _muon_plain(state)


def _orth_flops(rows, cols):
    m, n = min(rows, cols), max(rows, cols)
    # a step: the Gram matrix and its square (symmetric: one half each) and the product with X
    return 5 * (m * m * n + m * m * m + 2 * m * m * n)


def work(case):
    op = case["op"]
    if op == "lce":
        n, r, k, v = case["rows"], case["labelled"], case["hidden"], case["vocab"]
        nbytes = 2 * (r * k + v * k) + 8 * n + (4 * v if case["bias"] else 0)
        if not case["train"]:
            return {"bytes": nbytes + 4 * n, "flops": 2 * r * k * v}
        return {"bytes": nbytes + 2 * (n * k + v * k) + (4 * v if case["bias"] else 0) + 4, "flops": 6 * r * k * v}
    if op == "ffn":
        n, k, f = case["rows"], case["hidden"], case["inner"]
        if not case["train"]:
            return {"bytes": 2 * (2 * n * k + 3 * k * f), "flops": 6 * n * k * f}
        return {"bytes": 2 * (4 * n * k + 6 * k * f), "flops": 18 * n * k * f}
    if op == "orth":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": 2 * size * case["batch"] * case["rows"] * case["cols"],
                "flops": case["batch"] * _orth_flops(case["rows"], case["cols"])}
    shapes = _muon_shapes(case)
    # gradient, momentum and weight read, momentum and weight written
    return {"bytes": sum(20 * m * n for m, n in shapes), "flops": sum(_orth_flops(m, n) for m, n in shapes)}


def _lce_exact(case, seed):
    h, w, y, b, scale = _lce_inputs(case, seed)
    n, v = case["rows"], case["vocab"]
    w64 = w.double()
    rows = (y >= 0).nonzero().squeeze(1)
    loss = torch.zeros(n, dtype=torch.float64, device="cuda")
    dh = torch.zeros(n, case["hidden"], dtype=torch.float64, device="cuda")
    dw = torch.zeros_like(w64)
    db = torch.zeros(v, dtype=torch.float64, device="cuda")
    for part in rows.split(1024):
        hp, yp = h[part].double(), y[part]
        z = torch.mm(hp, w64.t().contiguous())
        if b is not None:
            z += b.double()
        logp = z - torch.logsumexp(z, dim=1, keepdim=True)
        pick = torch.zeros_like(z).scatter_(1, yp[:, None], 1.0)
        loss[part] = -(logp * pick).sum(dim=1)
        if case["train"]:
            dz = (logp.exp() - pick) * (scale / len(rows))
            dh[part] = torch.mm(dz, w64)
            dw += torch.mm(dz.t().contiguous(), hp)
            db += dz.sum(dim=0)
    if not case["train"]:
        return [loss]
    return [loss.sum() / len(rows), dh, dw] + ([db] if b is not None else [])


def _ffn_exact(case, seed):
    x, wg, wu, wd, dy = [None if t is None else t.double() for t in _ffn_inputs(case, seed)]
    outs, dwg, dwu, dwd = [], torch.zeros_like(wg), torch.zeros_like(wu), torch.zeros_like(wd)
    wgt, wut, wdt = (t.t().contiguous() for t in (wg, wu, wd))
    for i in range(0, len(x), 2048):
        xs = x[i:i + 2048]
        g, u = (torch.mm(xs, wgt).requires_grad_(case["train"]), torch.mm(xs, wut))
        act = {"silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid, "relu": torch.relu,
               "gelu": torch.nn.functional.gelu,
               "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[case["act"]]
        a = act(g)
        h = a.detach() * u
        y = torch.mm(h, wdt)
        if not case["train"]:
            outs.append((y,))
            continue
        dys = dy[i:i + 2048]
        dh = torch.mm(dys, wd)
        dg, = torch.autograd.grad(a, g, dh * u)
        du = dh * a.detach()
        outs.append((y, torch.mm(dg, wg) + torch.mm(du, wu)))
        dwg += torch.mm(dg.t().contiguous(), xs)
        dwu += torch.mm(du.t().contiguous(), xs)
        dwd += torch.mm(dys.t().contiguous(), h)
    cat = [torch.cat(t) for t in zip(*outs)]
    return cat + [dwg, dwu, dwd] if case["train"] else cat


def _orth_exact(x):
    """One matrix: X p(X^T X) with p(s) = a + b s + c s^2, from the side with the smaller Gram matrix."""
    a, b, c = _NS
    z = x.double()
    flip = z.shape[0] < z.shape[1]
    if flip:
        z = z.t().contiguous()
    z = z / (z.norm() + 1e-7)
    eye = torch.eye(z.shape[1], dtype=torch.float64, device=z.device)
    for _ in range(5):
        s = torch.mm(z.t().contiguous(), z)
        z = torch.mm(z, a * eye + torch.mm(s, b * eye + c * s))
    return z.t().contiguous() if flip else z


def exact(case, seed):
    op = case["op"]
    if op == "lce":
        return _lce_exact(case, seed)
    if op == "ffn":
        return _ffn_exact(case, seed)
    if op == "orth":
        return [torch.stack([_orth_exact(x) for x in _orth_inputs(case, seed)])]
    lr, mu, wd = _MUON["lr"], _MUON["momentum"], _MUON["weight_decay"]
    new_p, new_m = [], []
    for p, g, m in zip(*_muon_inputs(case, seed)):
        p, g = p.double(), g.double()
        m = mu * m.double() + g
        grow = math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        new_p.append((1.0 - lr * wd) * p - lr * grow * _orth_exact(g + mu * m))
        new_m.append(m)
    return new_p + new_m


