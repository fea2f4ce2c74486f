"""The transformer-step operators (linear_cross_entropy, gated_ffn, orthogonalize, Muon) on the GPU against
plain 64-bit formulas on the CPU.

Tolerances are worst-case bounds put together from the roundings that the kernels document: `u` is half a
step of the 16-bit type (bf16 2^-8 relative, fp16 2^-11), sums of n terms in fp32 are off by at most
n 2^-24 of the sum of magnitudes, exp and friends by 2^-18 relative.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
E32 = 2.0 ** -24
EXP = 2.0 ** -18


@pytest.fixture(scope="module", autouse=True)
def _kernels():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from mihvd import _native

    _native.require_kernels()


def half(dt):
    return torch.finfo(dt).eps / 2


def floor_of(dt):
    """Half the smallest step of the type (fp16 outputs below 6e-5 are subnormal)."""
    return 2.0 ** -25 if dt == FP else 0.0


def gen(seed):
    return torch.Generator().manual_seed(seed)


def close(got, want, tol, what):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol) & ~(torch.isnan(got) & torch.isnan(want))
    assert not bad.any(), "%s: %d of %d off, worst %.3g over %.3g" % (
        what, int(bad.sum()), bad.numel(), float((got - want).abs()[bad].max()),
        float((tol if torch.is_tensor(tol) else torch.tensor(tol)).expand_as(want)[bad].max()))


# ---------------------------------------------------------------------------------------------- #
# linear_cross_entropy


def lce_case(n, k, v, dt, bias, seed, drop=0.3):
    g = gen(seed)
    w = (torch.randn(v, k, generator=g, dtype=torch.float64) * 1.5 / math.sqrt(k)).to(dt)
    y = torch.randint(0, v, (n,), generator=g)
    h = (torch.randn(n, k, generator=g, dtype=torch.float64) + w.double()[y]).to(dt)
    y[torch.rand(n, generator=g) < drop] = -100
    b = None
    if bias is not None:
        b = (torch.randn(v, generator=g, dtype=torch.float64) * 0.3).to(bias)
    return h, w, y, b


def lce_ref(h, w, y, b, grow, dt):
    """Per-row loss, gradients for row weights `grow`, and their tolerances, in 64 bits."""
    h, w = h.double(), w.double()
    n, k = h.shape
    v = w.shape[0]
    u = half(dt)
    z = h @ w.t() + (0 if b is None else b.double())
    zerr = (k + 8) * E32 * (h.abs() @ w.abs().t() + (0 if b is None else b.double().abs())).max().item()
    keep = y != -100
    lse = torch.logsumexp(z, 1)
    safe = torch.where(keep, y, torch.zeros_like(y))
    loss = torch.where(keep, lse - z.gather(1, safe[:, None]).squeeze(1), torch.zeros_like(lse))
    rel = 2 * zerr + 2 * EXP + lse.abs().max().item() * 2.0 ** -22  # of a probability
    ltol = rel + loss.abs().max().item() * 2.0 ** -22
    p = torch.exp(z - lse[:, None])
    one = torch.zeros_like(z).scatter_(1, safe[:, None], 1.0)
    gk = (grow * keep)[:, None]
    dz = (p - one) * gk
    err = dz.abs() * (u + 2.0 ** -21) + p * gk.abs() * rel + 2.0 ** -38 * gk.abs().max()
    acc = dz.abs() + err
    dh = dz @ w
    dw = dz.t() @ h
    floor = floor_of(dt)
    dht = (err + acc * v * E32) @ w.abs() + dh.abs() * u + floor
    dwt = (err + acc * n * E32).t() @ h.abs() + dw.abs() * u + floor
    db = dz.sum(0)
    dbt = (p * gk.abs() * rel + dz.abs() * (n + 8) * E32).sum(0) + db.abs() * (u if b is not None and b.dtype == dt else
                                                                             2.0 ** -22) + 1e-12 + floor
    return loss, ltol, (dh, dht), (dw, dwt), (db, dbt)


LCE = [  # rows, hidden, vocabulary
    (1, 8, 1), (1, 768, 1000), (5, 17, 33), (20, 64, 257), (127, 100, 511), (130, 72, 1025), (300, 200, 130),
    (257, 333, 777),
]


@pytest.mark.parametrize("dt", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("n,k,v", LCE)
def test_lce_mean_and_gradients(n, k, v, dt):
    from mihvd.ops import linear_cross_entropy

    h, w, y, b = lce_case(n, k, v, dt, torch.float32 if v % 2 else dt, seed=n + k + v)
    if (y == -100).all():
        y[0] = 0
    scale = 1024.0 if dt == FP else 1.0
    cnt = int((y != -100).sum())
    loss, ltol, dh, dw, db = lce_ref(h, w, y, b, torch.full((n,), scale / cnt, dtype=torch.float64), dt)
    leaves = [t.cuda().requires_grad_() for t in (h, w, b)]
    out = linear_cross_entropy(leaves[0], leaves[1], y.cuda(), leaves[2])
    assert out.dtype == torch.float32 and out.shape == ()
    close(out, loss.sum() / cnt, ltol + n * E32 * float(loss.abs().max()), "loss")
    gh, gw, gb = torch.autograd.grad(out, leaves, torch.tensor(scale, device="cuda"))
    assert (gh.dtype, gw.dtype, gb.dtype) == (dt, dt, b.dtype)
    close(gh, *dh, "dh")
    close(gw, *dw, "dw")
    close(gb, *db, "db")
    assert (gh.cpu()[y == -100] == 0).all()


@pytest.mark.parametrize("dt", [BF, FP], ids=["bf16", "fp16"])
def test_lce_none_with_row_weights_and_sum(dt):
    from mihvd.ops import linear_cross_entropy

    n, k, v = 150, 96, 300
    h, w, y, _ = lce_case(n, k, v, dt, None, seed=3)
    grow = torch.randn(n, generator=gen(5), dtype=torch.float64).float().double() * 16
    grow[7] = 0
    loss, ltol, dh, dw, _ = lce_ref(h, w, y, None, grow, dt)
    hl, wl = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    rows = linear_cross_entropy(hl.view(3, 50, k), wl, y.cuda().view(3, 50), reduction="none")
    assert rows.shape == (3, 50)
    close(rows.reshape(-1), loss, ltol, "rows")
    gh, gw = torch.autograd.grad(rows, [hl, wl], grow.float().cuda().view(3, 50))
    close(gh, *dh, "dh")
    close(gw, *dw, "dw")
    total = linear_cross_entropy(hl, wl, y.cuda(), reduction="sum")
    close(total, loss.sum(), n * ltol + n * E32 * float(loss.sum()), "sum")
    ones = lce_ref(h, w, y, None, torch.ones(n, dtype=torch.float64), dt)
    gh, gw = torch.autograd.grad(total, [hl, wl])
    close(gh, *ones[2], "dh of the sum")
    close(gw, *ones[3], "dw of the sum")


def test_lce_masked_vocabulary_and_bad_rows():
    """Bias entries of -inf and of the type's lowest value leave their words out; nothing labelled; a label
    outside the vocabulary poisons its own row; NaN in an ignored row stays there."""
    from mihvd.ops import linear_cross_entropy

    n, k, v = 40, 64, 300
    h, w, y, b = lce_case(n, k, v, BF, torch.float32, seed=11)
    off = torch.arange(v) % 3 == 1
    y = torch.where((y >= 0) & off[y.clamp(min=0)], y - 1, y)
    for low in (-math.inf, torch.finfo(torch.float32).min):
        b[off] = low
        cnt = int((y != -100).sum())
        bb = b.double().masked_fill(off, -math.inf)
        z = h.double() @ w.double().t() + bb
        want = torch.nn.functional.cross_entropy(z, y)
        leaves = [h.cuda().requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()]
        out = linear_cross_entropy(leaves[0], leaves[1], y.cuda(), leaves[2])
        close(out, want, 1e-4, "loss")
        gh, gw, gb = torch.autograd.grad(out, leaves)
        assert torch.isfinite(gh).all() and torch.isfinite(gw).all()
        assert (gw.cpu()[off] == 0).all() and (gb.cpu()[off] == 0).all()
    none = torch.full((n,), -100, device="cuda")
    out = linear_cross_entropy(leaves[0], leaves[1], none)
    assert torch.isnan(out)
    gh, gw = torch.autograd.grad(out, leaves[:2])
    assert (gh == 0).all() and (gw == 0).all()
    hn = h.clone()
    hn[y == -100] = math.nan
    out = linear_cross_entropy(hn.cuda(), leaves[1], y.cuda(), reduction="none")
    assert torch.isfinite(out).all()
    yb = y.clone()
    yb[y != -100] = torch.where(torch.arange(cnt) == 2, torch.tensor(v), yb[y != -100])
    out = linear_cross_entropy(h.cuda(), leaves[1], yb.cuda(), reduction="none").cpu()
    assert torch.isnan(out[yb == v]).all() and torch.isfinite(out[yb != v]).all()


def test_lce_strides_and_empty():
    """Transposed and sliced operands; no rows at all; another ignore_index."""
    from mihvd.ops import linear_cross_entropy

    n, k, v = 70, 40, 200
    h, w, y, _ = lce_case(n, k, v, BF, None, seed=21)
    wide = torch.zeros(n, k + 24, dtype=BF, device="cuda")
    wide[:, 8:8 + k] = h.cuda()
    odd = torch.zeros(n, k + 3, dtype=BF, device="cuda")
    odd[:, 3:] = h.cuda()
    plain = [h.cuda().requires_grad_(), w.cuda().requires_grad_()]
    base = linear_cross_entropy(*plain, y.cuda())
    want = torch.autograd.grad(base, plain)
    for hv in (wide[:, 8:8 + k], odd[:, 3:], h.cuda().t().contiguous().t()):
        for wv in (w.cuda(), w.cuda().t().contiguous().t()):
            hl, wl = hv.detach().requires_grad_(), wv.detach().requires_grad_()
            out = linear_cross_entropy(hl, wl, y.cuda())
            assert torch.equal(out, base)
            gh, gw = torch.autograd.grad(out, [hl, wl])
            assert all(torch.equal(a, b) for a, b in zip((gh, gw), want))
    e = linear_cross_entropy(torch.empty(0, k, dtype=BF, device="cuda"), w.cuda(), torch.empty(0, dtype=torch.long,
                                                                                             device="cuda"), reduction="sum")
    assert float(e) == 0
    y2 = y.clone()
    y2[y == -100] = 7
    a = linear_cross_entropy(h.cuda(), w.cuda(), y2.cuda(), ignore_index=7)
    y3 = torch.where(y2 == 7, torch.tensor(-100), y2)
    assert torch.equal(a, linear_cross_entropy(h.cuda(), w.cuda(), y3.cuda()))


# ---------------------------------------------------------------------------------------------- #
# gated_ffn


def act64(name, g):
    g = g.detach().requires_grad_()
    f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "sigmoid": torch.sigmoid,
         "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[name]
    a = f(g)
    d, = torch.autograd.grad(a.sum(), g)
    return a.detach(), d


def ffn_ref(x, wg, wu, wd, dy, act, dt):
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    n, k = x.shape
    f = wg.shape[0]
    r = half(dt)
    lo = floor_of(dt)
    g, u = x @ wg.t(), x @ wu.t()
    ge, ue = (k + 2) * E32 * (x.abs() @ wg.abs().t()), (k + 2) * E32 * (x.abs() @ wu.abs().t())
    a, d = act64(act, g)
    h = a * u
    # activations have |act'| <= 1.13 and, away from relu's corner, |act''| <= 0.8; the functions of
    # exp, erf and tanh are off by EXP of their argument's size
    ae = 1.13 * ge + EXP * (1 + g.abs())
    he = ae * u.abs() + (a.abs() + ae) * ue + r * h.abs() + lo
    y = h @ wd.t()
    ye = (he + (h.abs() + he) * (f + 2) * E32) @ wd.abs().t() + r * y.abs() + lo
    # backward: g and u rounded to 16 bits
    gr, ur = ge + r * g.abs() + lo, ue + r * u.abs() + lo
    dh = dy @ wd
    dhe = (k + 2) * E32 * (dy.abs() @ wd.abs())
    de = 0.8 * gr + EXP * (1 + g.abs())
    if act == "relu":
        de = torch.where(g.abs() <= gr, torch.ones_like(g), torch.zeros_like(g))
    are = 1.13 * gr + EXP * (1 + g.abs())
    dg, du = dh * u * d, dh * a
    dge = (dh.abs() + dhe) * ((u.abs() + ur) * (d.abs() + de) - u.abs() * d.abs()) + dhe * u.abs() * d.abs()
    dge = dge + r * (dg.abs() + dge) + lo
    due = (dh.abs() + dhe) * are + dhe * a.abs()
    due = due + r * (du.abs() + due) + lo

    def mm(p, pe, q, terms):  # p @ q with p off by pe, rounded once
        out = p @ q
        return out, (pe + (p.abs() + pe) * (terms + 2) * E32) @ q.abs() + r * out.abs() * 1.01 + lo

    dx1, dx1e = mm(dg, dge, wg, 2 * f)
    dx2, dx2e = mm(du, due, wu, 2 * f)
    return [(y, ye), (dx1 + dx2, dx1e + dx2e), mm(dg.t(), dge.t(), x, n), mm(du.t(), due.t(), x, n),
            mm(dy.t(), torch.zeros_like(dy.t()), h, n)[:1] + ((dy.abs().t() @ (he + (h.abs() + he) * (n + 2) * E32))
                                                          + r * (dy.t() @ h).abs() * 1.01 + lo,)]


def ffn_case(n, k, f, dt, seed):
    g = gen(seed)

    def r(*s, by=1.0):
        return (torch.randn(*s, generator=g, dtype=torch.float64) * by).to(dt)

    return r(n, k), r(f, k, by=k ** -0.5), r(f, k, by=k ** -0.5), r(k, f, by=f ** -0.5), r(n, k)


FFN = [(1, 8, 8), (1, 768, 2048), (3, 17, 5), (17, 96, 130), (64, 64, 64), (129, 130, 257), (200, 264, 72), (513, 40, 136)]


@pytest.mark.parametrize("dt", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("n,k,f", FFN)
def test_ffn_forward_and_gradients(n, k, f, dt):
    from mihvd.ops import gated_ffn
    from mihvd.ops.transformer import ACTIVATIONS

    acts = ACTIVATIONS if n == 17 else [ACTIVATIONS[(n + k) % len(ACTIVATIONS)]]
    x, wg, wu, wd, dy = ffn_case(n, k, f, dt, n + k + f)
    for act in acts:
        want = ffn_ref(x, wg, wu, wd, dy, act, dt)
        leaves = [t.cuda().requires_grad_() for t in (x, wg, wu, wd)]
        y = gated_ffn(*leaves, activation=act)
        close(y, *want[0], act + " y")
        with torch.no_grad():
            assert torch.equal(gated_ffn(*leaves, activation=act), y)
        for got, ref, name in zip(torch.autograd.grad(y, leaves, dy.cuda()), want[1:], ("dx", "dwg", "dwu", "dwd")):
            assert got.dtype == dt
            close(got, *ref, act + " " + name)


def test_ffn_partial_gradients_strides_and_shapes():
    from mihvd.ops import gated_ffn

    x, wg, wu, wd, dy = (t.cuda() for t in ffn_case(48, 64, 96, BF, 9))
    full = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    want = torch.autograd.grad(gated_ffn(*full), full, dy)
    for on in range(4):
        part = [t.clone().requires_grad_(i == on) for i, t in enumerate((x, wg, wu, wd))]
        got, = torch.autograd.grad(gated_ffn(*part), [part[on]], dy)
        assert torch.equal(got, want[on]), on
    packed = torch.cat([wg, wu]).contiguous()
    views = [x.view(2, 4, 6, 64).transpose(0, 1), packed[:96], packed[96:], wd.t().contiguous().t()]
    views = [t.detach().requires_grad_() for t in views]
    y = gated_ffn(*views)
    ref = gated_ffn(x, wg, wu, wd)
    assert torch.equal(y, ref.view(2, 4, 6, 64).transpose(0, 1))
    got = torch.autograd.grad(y, views, dy.view(2, 4, 6, 64).transpose(0, 1))
    # the rows come in another order: the sums over rows differ by their rounding only
    assert torch.equal(got[0], want[0].view(2, 4, 6, 64).transpose(0, 1))
    for a, b in zip(got[1:], want[1:]):
        assert (a.float() - b.float()).abs().max() <= 2 ** -7 * b.float().abs().max()
    assert gated_ffn(x[:0], wg, wu, wd).shape == (0, 64)


# ---------------------------------------------------------------------------------------------- #
# orthogonalize and Muon

NS_SHAPES = [(1, 1), (1, 7), (9, 1), (8, 8), (17, 33), (64, 64), (130, 65), (65, 200), (256, 136), (128, 300)]


def ns64(x, steps=5, coef=(3.4445, -4.7750, 2.0315), eps=1e-7):
    a, b, c = coef
    z = x.double()
    z = z / (torch.linalg.vector_norm(z, dim=(-2, -1), keepdim=True) + eps)
    for _ in range(steps):
        s = z @ z.transpose(-2, -1)
        z = a * z + (b * s + c * (s @ s)) @ z
    return z


def ns_tol(want, out_dt, split):
    """Relative to the Frobenius norm: six matrices of up to three roundings each, an error growing by at
    most a factor of five relative to the values in the steps that follow (|f'(s)| s / |f(s)| <= 5 on the
    singular values' range): below 90 / sqrt(3) < 64 half steps of the planes; then the output's own."""
    step = 2.0 ** -22 if split else 2.0 ** -11
    return (64 * step + half(out_dt)) * torch.linalg.vector_norm(want).item()


@pytest.mark.parametrize("dt", [torch.float32, BF, FP], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("m,n", NS_SHAPES)
def test_orthogonalize(m, n, dt):
    from mihvd.optim import orthogonalize

    g = gen(m * 1000 + n)
    x = (torch.randn(3, m, n, generator=g, dtype=torch.float64) * 1e-2).to(dt)
    x[1] = (x[1].double() * 1e-3).to(dt) if dt != FP else x[1]
    got = orthogonalize(x.cuda())
    assert got.dtype == dt and got.shape == x.shape
    for i in range(3):
        want = ns64(x[i])
        err = torch.linalg.vector_norm(got[i].double().cpu() - want).item()
        assert err <= ns_tol(want, dt, dt == torch.float32), (i, err, ns_tol(want, dt, dt == torch.float32))
    assert torch.equal(orthogonalize(x[2].cuda()), got[2])  # alone or in a batch


def test_orthogonalize_edges():
    from mihvd.optim import orthogonalize

    z = torch.zeros(5, 9, device="cuda")
    assert (orthogonalize(z) == 0).all()
    x = torch.randn(40, 24, generator=gen(1)).cuda()
    assert torch.isnan(orthogonalize(torch.where(torch.arange(24, device="cuda") == 3, math.nan, x))).all()
    s = orthogonalize(x, steps=0)
    close(s, x.cpu().double() / x.cpu().double().norm(), 2.0 ** -20, "normalised")
    one = orthogonalize(x, steps=1)
    w1 = ns64(x.cpu(), 1)
    assert torch.linalg.vector_norm(one.double().cpu() - w1) <= ns_tol(w1, torch.float32, True)
    coarse = orthogonalize(x, precision="fp16")
    w5 = ns64(x.cpu())
    assert coarse.dtype == torch.float32
    assert torch.linalg.vector_norm(coarse.double().cpu() - w5) <= ns_tol(w5, torch.float32, False)
    t = torch.randn(24, 40, generator=gen(2)).cuda().t()
    assert torch.equal(orthogonalize(t), orthogonalize(t.contiguous()))
    many = torch.randn(35, 6, 10, generator=gen(3)).cuda()
    assert torch.equal(orthogonalize(many)[33], orthogonalize(many[33]))
    assert orthogonalize(many[:0]).shape == (0, 6, 10)
    assert orthogonalize(many.view(5, 7, 6, 10)).shape == (5, 7, 6, 10)


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("scale", ["spectral", "rms"])
def test_muon_steps(nesterov, scale):
    from mihvd.optim import Muon

    g = gen(17)
    shapes = [(24, 40), (24, 40), (50, 16), (8, 3, 5, 5), (24, 40)]
    ps = [torch.randn(*s, generator=g) * 0.1 for s in shapes]
    params = [torch.nn.Parameter(p.cuda()) for p in ps]
    opt = Muon(params, lr=0.03, momentum=0.9, nesterov=nesterov, weight_decay=0.1, scale=scale)
    ref = [p.double() for p in ps]
    mom = [torch.zeros_like(p) for p in ref]
    for _ in range(3):
        grads = [torch.randn(*s, generator=g) * 1e-2 for s in shapes]
        for p, d in zip(params, grads):
            p.grad = d.cuda()
        params[2].grad = None  # no gradient: the parameter and its momentum stay
        opt.step()
        for i, d in enumerate(grads):
            if i == 2:
                continue
            mom[i] = 0.9 * mom[i] + d.double()
            u = d.double() + 0.9 * mom[i] if nesterov else mom[i]
            r, c = shapes[i][0], ref[i].numel() // shapes[i][0]
            s = math.sqrt(max(1.0, r / c)) if scale == "spectral" else 0.2 * math.sqrt(max(r, c))
            o = ns64(u.reshape(r, c))
            ref[i] = ref[i] * (1 - 0.03 * 0.1) - 0.03 * s * o.view(shapes[i])
    for i in range(len(shapes)):
        want = ref[i]
        # three steps; momentum in fp32 is off by 2^-22 of its size, the update by ns_tol's 64 * 2^-22
        tol = 3 * (2.0 ** -22 * float(want.norm()) + 0.03 * 8 * 128 * 2.0 ** -22 * math.sqrt(min(shapes[i][0], 1e9)))
        assert float((params[i].detach().double().cpu() - want).norm()) <= tol, i
        if i != 2:
            m = opt.state[params[i]]["momentum_buffer"].double().cpu()
            assert float((m - mom[i]).norm()) <= 8 * 2.0 ** -24 * float(mom[i].norm()) + 1e-12


def test_muon_other_types_and_layouts():
    """bf16 parameters and channels_last weights take torch operations around the same products."""
    from mihvd.optim import Muon

    g = gen(23)
    w = torch.randn(32, 8, 3, 3, generator=g)
    d = torch.randn(32, 8, 3, 3, generator=g) * 1e-2
    a = torch.nn.Parameter(w.cuda())
    b = torch.nn.Parameter(w.cuda().to(memory_format=torch.channels_last))
    for p in (a, b):
        p.grad = d.cuda() if p is a else d.cuda().to(memory_format=torch.channels_last)
        Muon([p], lr=0.1, weight_decay=0.1).step()
    assert (a - b).abs().max() <= 2.0 ** -20 * a.abs().max()
    c = torch.nn.Parameter(w.cuda().bfloat16())
    c.grad = d.cuda().bfloat16()
    Muon([c], lr=0.1, weight_decay=0.1).step()
    assert (a - c.float()).abs().max() <= 2.0 ** -6 * a.abs().max()
