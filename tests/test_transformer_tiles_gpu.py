"""The transformer-step operators at sizes that reach every tile, split and piece of their products, against the
formulas in 64 bits (in elementary operations on the GPU, where the CPU would take minutes). Each case names
the plan that it is there for; on a GPU of 256 compute units the plan has to be that one."""
import math

import pytest
import torch

from test_transformer_gpu import BF, E32, FP, close, ffn_case, ffn_ref, gen, lce_case, lce_ref, ns64, ns_tol

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _kernels():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from mihvd import _native

    _native.require_kernels()
    yield
    torch.cuda.empty_cache()


def planned(op, sizes, want):
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert list(torch.ops.mihvd.transformer_plan(op, sizes)) == want


def near(got, pair, what):
    close(got, pair[0].cpu(), pair[1].cpu() if torch.is_tensor(pair[1]) else pair[1], what)


# rows, hidden, vocabulary, type, bias; tiles of the logits, dz, dh, dW; dh's splits at most; pieces
LCE = [
    (1300, 200, 30522, BF, None, [256, 256, 128, 128, 23, 1]),      # several output tiles a block, a k tile that ends inside
    (1300, 200, 30522, FP, torch.float32, [256, 128, 128, 128, 23, 1]),  # the bias gradient over several row tiles
    (3000, 700, 12000, BF, BF, [256, 128, 128, 256, 3, 1]),         # eleven k tiles
    (8200, 200, 33100, BF, torch.float32, [256, 128, 256, 128, 7, 2]),   # two pieces, a short ragged one last
    (8200, 136, 33100, FP, None, [256, 256, 256, 128, 7, 2]),
    (8925, 1021, 106, BF, torch.float32, [64, 64, 256, 64, 1, 1]),  # dh at 256 without splits
    (65, 129, 39157, FP, None, [128, 128, 64, 256, 41, 1]),
]


@pytest.mark.parametrize("n,k,v,dt,bias,plan", LCE, ids=["%dx%dx%d" % c[:3] + ("-bias" if c[4] else "") for c in LCE])
def test_lce_tiles(n, k, v, dt, bias, plan):
    from mihvd.ops import linear_cross_entropy

    planned("linear_cross_entropy", [n, k, v, int(bias is not None)], plan)
    h, w, y, b = lce_case(n, k, v, dt, bias, seed=n + k)
    y[-1] = v - 1
    y[-2] = 0
    cnt = int((y != -100).sum())
    scale = 4096.0 if dt == FP else 1.0
    dev = [t if t is None else t.cuda() for t in (h, w, y, b)]
    grow = torch.full((n,), scale / cnt, dtype=torch.float64, device="cuda")
    loss, ltol, dh, dw, db = lce_ref(*dev, grow, dt)
    leaves = [t.requires_grad_() for t in (dev[0], dev[1], dev[3]) if t is not None]
    out = linear_cross_entropy(dev[0], dev[1], dev[2], dev[3])
    near(out, (loss.sum() / cnt, ltol + n * E32 * float(loss.abs().max())), "loss")
    grads = torch.autograd.grad(out, leaves, torch.tensor(scale, device="cuda"))
    for got, ref, name in zip(grads, (dh, dw, db), ("dh", "dw", "db")):
        near(got, ref, name)
    assert (grads[0][dev[2] == -100] == 0).all()
    # worst-case bounds grow with the number of terms; taken together errors are a rounding of dz and one of the
    # result, each off by half a step at most: within twice that of the norm
    for got, ref, name in zip(grads[:2], (dh, dw), ("dh", "dw")):
        err = torch.linalg.vector_norm(got.double() - ref[0]) / torch.linalg.vector_norm(ref[0])
        assert float(err) <= 2 * torch.finfo(dt).eps / 2, (name, float(err))
    with torch.no_grad():
        rows = linear_cross_entropy(dev[0], dev[1], dev[2], dev[3], reduction="none")
    near(rows, (loss, ltol), "rows")


# rows, hidden, inner; the gate product's tile; tile and splits of y, dWd, dWg and dWu, dx
FFN = [
    (2100, 1032, 4100, BF, "silu", [128, 128, 3, 128, 1, 256, 1, 128, 3]),
    (9000, 264, 5000, BF, "gelu", [256, 128, 1, 128, 4, 128, 2, 128, 2]),
    (10925, 147, 2520, FP, "gelu_tanh", [256, 128, 1, 128, 12, 128, 6, 256, 5]),
    (9773, 796, 66, BF, "sigmoid", [128, 256, 1, 64, 9, 64, 9, 256, 1]),
    (12511, 131, 5504, BF, "silu", [256, 256, 5, 128, 5, 256, 5, 256, 5]),
    (70, 648, 5504, FP, "silu", [128, 64, 11, 64, 1, 256, 1, 64, 11]),
    (66, 1539, 5664, BF, "gelu", [128, 64, 5, 256, 1, 128, 1, 64, 5]),
    (7161, 416, 5808, FP, "silu", [256, 128, 1, 256, 5, 128, 1, 256, 4]),
]


@pytest.mark.parametrize("n,k,f,dt,act,plan", FFN, ids=["%dx%dx%d" % c[:3] for c in FFN])
def test_ffn_tiles(n, k, f, dt, act, plan):
    from mihvd.ops import gated_ffn

    planned("gated_ffn", [n, k, f], plan)
    dev = [t.cuda() for t in ffn_case(n, k, f, dt, n + f)]
    want = ffn_ref(*dev, act, dt)
    leaves = [t.requires_grad_() for t in dev[:4]]
    y = gated_ffn(*leaves, activation=act)
    near(y, want[0], "y")
    grads = torch.autograd.grad(y, leaves, dev[4])
    for got, ref, name in zip(grads, want[1:], ("dx", "dwg", "dwu", "dwd")):
        near(got, ref, name)
    # as above: the kept projections' rounding, that of dg or du (twice through the product) and the result's
    for got, ref, name in zip((y, *grads), want, ("y", "dx", "dwg", "dwu", "dwd")):
        err = torch.linalg.vector_norm(got.detach().double() - ref[0]) / torch.linalg.vector_norm(ref[0])
        assert float(err) <= 4 * torch.finfo(dt).eps / 2, (name, float(err))


# matrices, rows, columns, planes; tiles of X X^T, the polynomial, X's update, the last update
NS = [
    (12, 575, 530, 1, [128, 128, 128, 128]), (12, 516, 648, 1, [128, 128, 128, 128]),
    (12, 575, 530, 2, [128, 128, 64, 64]), (12, 516, 648, 2, [128, 128, 64, 64]),
    (10, 1198, 1222, 1, [256, 128, 256, 128]), (11, 1254, 1165, 1, [256, 128, 128, 128]),
    (9, 3940, 66, 1, [64, 64, 128, 128]), (10, 3582, 131, 1, [64, 64, 256, 64]),
    (10, 1653, 65, 2, [64, 64, 128, 128]), (6, 65, 2800, 2, [64, 64, 128, 128]), (3, 2100, 2500, 2, [128, 128, 128, 128]),
]


def ns_wide(x, **kw):
    return ns64(x.transpose(-2, -1), **kw).transpose(-2, -1) if x.shape[-2] > x.shape[-1] else ns64(x, **kw)


@pytest.mark.parametrize("b,m,n,planes,plan", NS, ids=["%dx%dx%d-%d" % c[:4] for c in NS])
def test_orthogonalize_tiles(b, m, n, planes, plan):
    from mihvd.optim import orthogonalize

    planned("orthogonalize", [b, m, n, planes], plan)
    x = (torch.randn(b, m, n, generator=torch.Generator("cuda").manual_seed(m + n), device="cuda") * 1e-2)
    for dt in ((torch.float32,) if planes == 2 else (BF, FP, torch.float32)):
        xd = x.to(dt)
        got = orthogonalize(xd, precision="fp32" if planes == 2 else "fp16")
        want = ns_wide(xd)
        for i in range(b):
            err = torch.linalg.vector_norm(got[i].double() - want[i]).item()
            assert err <= ns_tol(want[i], dt, planes == 2), (dt, i, err)


def test_muon_tiles():
    """Ragged groups whose updates run at 128, straight and turned, with the weights' update in their epilogue."""
    from mihvd.optim import Muon

    shapes = [(1653, 65)] * 6 + [(65, 2800)] * 6 + [(100, 900)] * 3 + [(2100, 2500)] * 2 + [(2048, 2300)]
    g = torch.Generator("cuda").manual_seed(9)
    params = [torch.nn.Parameter(torch.randn(*s, generator=g, device="cuda") * 0.02) for s in shapes]
    start = [p.detach().double() for p in params]
    opt = Muon(params, lr=0.02, weight_decay=0.1)
    grads = [torch.randn(*s, generator=g, device="cuda") * 1e-2 for s in shapes]
    for p, d in zip(params, grads):
        p.grad = d
    opt.step()
    for i, (p, d) in enumerate(zip(params, grads)):
        r, c = shapes[i]
        o = ns_wide(d.double() * 1.95) * math.sqrt(max(1.0, r / c))
        want = start[i] * (1 - 0.02 * 0.1) - 0.02 * o
        tol = 0.02 * ns_tol(o, torch.float32, True) + 4 * E32 * float(torch.linalg.vector_norm(want))
        assert float(torch.linalg.vector_norm(p.detach().double() - want)) <= tol, i
        m = opt.state[p]["momentum_buffer"]
        assert torch.equal(m, d)


@pytest.mark.parametrize("precision", ["fp32", "fp16"])
def test_muon_without_steps(precision):
    """ns_steps=0: the update is the normalised momentum itself."""
    from mihvd.optim import Muon

    shapes = [(24, 40), (50, 16), (130, 257), (1, 9)]
    g = gen(19)
    ps, ds = ([torch.randn(*s, generator=g) for s in shapes] for _ in range(2))
    params = [torch.nn.Parameter(p.cuda()) for p in ps]
    for p, d in zip(params, ds):
        p.grad = d.cuda()
    Muon(params, lr=0.5, ns_steps=0, weight_decay=0.1, momentum=0.5, precision=precision).step()
    for p, w, d, (r, c) in zip(params, ps, ds, shapes):
        o = d.double() / (torch.linalg.vector_norm(d.double()) + 1e-7 / 1.5) * math.sqrt(max(1.0, r / c))
        want = w.double() * (1 - 0.05) - 0.5 * o
        # X rounded to its planes (22 or 11 bits of each value, 2^-37 at the least), the weight twice
        tol = 0.5 * (o.abs() * 2.0 ** (-22 if precision == "fp32" else -11) + 2.0 ** -36) + 4 * E32 * (w.double().abs() + 1)
        close(p, want, tol, "p")
