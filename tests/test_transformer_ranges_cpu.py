"""The optimizer side of the transformer-step operators at the ends of their ranges, without a GPU."""
import copy
import math

import pytest
import torch

from test_transformer_cpu import ns64


def muon_drift(dt, device, steps=40):
    """A 16-bit parameter through many steps of one small gradient with noise, beside the 64-bit recurrence over
    the same gradients: the largest error of the momentum, relative to its own size, and of the weight in
    half steps of its type per step."""
    from mihvd.optim import Muon

    g = torch.Generator().manual_seed(5)
    start = (torch.randn(24, 16, generator=g) * 0.5).to(dt)
    drift = torch.randn(24, 16, generator=g) * 2e-3
    w = torch.nn.Parameter(start.to(device))
    opt = Muon([w], lr=0.02, momentum=0.99, weight_decay=0.01)
    ref, mom = start.double(), torch.zeros(24, 16, dtype=torch.float64)
    for k in range(steps):
        d = ((torch.randn(24, 16, generator=g) * (0.3 if k == 0 else 1e-3)) + drift).to(dt)
        w.grad = d.to(device)
        opt.step()
        mom = 0.99 * mom + d.double()
        u = d.double() + 0.99 * mom
        ref = ref * (1 - 0.02 * 0.01) - 0.02 * math.sqrt(24 / 16) * ns64(u.t()).t()
    got = opt.state[w]["momentum_buffer"]
    assert got.dtype == torch.float32
    assert float((got.cpu().double() - mom).abs().max()) <= 2 * steps * 2.0 ** -24 * float(mom.abs().max())
    # each step rounds the weight once; the updates' own errors (ns_tol: 64 * 2^-22 of their norm) are far below
    half = torch.finfo(dt).eps / 2
    tol = steps * (half * (float(ref.abs().max()) + 0.5) + 0.02 * 1.3 * 6 * 64 * 2.0 ** -22)
    assert float((w.detach().cpu().double() - ref).abs().max()) <= tol


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_muon_momentum_of_16_bit_parameters(dt):
    muon_drift(dt, "cpu")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
def test_muon_checkpoint_keeps_the_momentum(dt):
    """A momentum goes through state_dict and load_state_dict bit for bit, and the step behind it is the same."""
    from mihvd.optim import Muon

    g = torch.Generator().manual_seed(6)
    a = [torch.nn.Parameter(torch.randn(6, 4, generator=g).to(dt)) for _ in range(3)]
    opt = Muon([dict(params=a[:1]), dict(params=a[1:], lr=0.05)], lr=0.02)
    for k in range(3):
        for i, p in enumerate(a):
            p.grad = None if i == 1 and k == 0 else (torch.randn(6, 4, generator=g) * 0.1).to(dt)
        opt.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    opt2 = Muon([dict(params=b[:1]), dict(params=b[1:])], lr=0.02)
    opt2.load_state_dict(copy.deepcopy(opt.state_dict()))
    for p, q in zip(a, b):
        m, n = opt.state[p]["momentum_buffer"], opt2.state[q]["momentum_buffer"]
        assert m.dtype == n.dtype == torch.float32 and torch.equal(m, n)
        q.grad = p.grad.clone()
    opt.step()
    opt2.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    # a checkpoint that holds the momentum in the parameter's type loads into fp32
    old = copy.deepcopy(opt.state_dict())
    for st in old["state"].values():
        st["momentum_buffer"] = st["momentum_buffer"].to(dt)
    opt2.load_state_dict(old)
    assert all(opt2.state[q]["momentum_buffer"].dtype == torch.float32 for q in b)


@pytest.mark.parametrize("steps,coef", [(1, (3.4445, -4.7750, 2.0315)), (5, (3.4445, -4.7750, 2.0315)),
                                        (100, (3.4445, -4.7750, 2.0315)), (100, (1.5, -0.5, 0.0)), (7, (2.0, -1.5, 0.5)),
                                        (3, (4.0, -2.0, 1.0)), (2, (-3.0, 0.0, 0.0)), (4, (3.0, 0.0, 0.0)), (3, (0.0, 4.0, -1.0)),
                                        (3, (1.0, 2.0, -2.5)), (0, (9.0, 0.0, 0.0)), (3, (0.0, 0.0, 0.0))])
def test_newton_schulz_reach(steps, coef):
    """The bound on X, X X^T and the polynomial is what a fine grid of singular values attains."""
    from mihvd.optim import _ns_reach

    a, b, c = coef
    lo, hi, want = 0.0, 1.0, 1.0
    for _ in range(steps):
        s = torch.linspace(lo, hi, 400001, dtype=torch.float64)
        t = s * s
        q = a + b * t + c * t * t
        want = max(want, hi, hi * hi, float(q.abs().max()))
        hi = float((s * q).abs().max())
        if want > 1e9:
            break
    got = _ns_reach(steps, a, b, c)
    assert want <= got * (1 + 1e-12) and (got <= want * (1 + 1e-6) or want > 1e9), (got, want)


def test_muon_group_options():
    """A group's own options are checked as the constructor's are, when it is added, loaded, or has been edited."""
    from mihvd.optim import Muon

    def par():
        return torch.nn.Parameter(torch.ones(4, 3))

    bad = (dict(lr=-1.0), dict(momentum=1.5), dict(weight_decay=-1.0), dict(ns_steps=101), dict(ns_steps=-1), dict(scale="adam"),
           dict(precision="bf16"), dict(ns_coefficients=(1.0, 2.0)), dict(ns_coefficients=(16.0, 0.0, 0.0)))
    opt = Muon([par()])
    for kw in bad:
        with pytest.raises(ValueError, match="Muon"):
            Muon([dict(params=[par()], **kw)])
        with pytest.raises(ValueError, match="Muon"):
            opt.add_param_group(dict(params=[par()], **kw))
        assert len(opt.param_groups) == 1
        state = copy.deepcopy(opt.state_dict())
        state["param_groups"][0].update(kw)
        with pytest.raises(ValueError, match="Muon"):
            opt.load_state_dict(state)
        assert opt.param_groups[0]["scale"] == "spectral" and opt.param_groups[0]["ns_steps"] == 5
        other = Muon([par(), par()])
        other.param_groups[0].update(kw)
        p = other.param_groups[0]["params"][0]
        p.grad = torch.ones(4, 3)
        with pytest.raises(ValueError, match="Muon"):
            other.step()
        assert (p == 1).all() and not other.state
    opt.add_param_group(dict(params=[par()], ns_steps=3, scale="rms", precision="fp16", ns_coefficients=[1.5, -0.5, 0]))
    assert opt.param_groups[1]["ns_coefficients"] == (1.5, -0.5, 0.0)


@pytest.mark.parametrize("by,eps", [(2.0 ** 100, 1e-7), (2.0 ** 120, 1e-7), (2.0 ** -90, 0.0)])
def test_orthogonalize_far_norms_cpu(by, eps):
    """Values whose squares leave fp32's range have the result of their moderate multiple."""
    from mihvd.optim import orthogonalize

    x = torch.randn(12, 7, generator=torch.Generator().manual_seed(8))
    want = ns64(x, eps=0.0)
    got = orthogonalize(x * by, eps=eps)
    assert float((got.double() - want).norm()) <= 64 * 5 * 2.0 ** -24 * float(want.norm())


def _plan(op, *sizes):
    from mihvd import _native

    if not _native.load_kernels():
        pytest.skip("no kernel library")
    return list(torch.ops.mihvd.transformer_plan(op, list(sizes)))


def _estimate(tile, m, n, k, epi=1.0, batch=1, cus=256):
    """us of an unsplit product, by the measured terms that the plan names."""
    tiles = -(-m // tile) * -(-n // tile) * batch
    two = tile < 256 and tiles > cus
    unit = {256: 1.45, 128: 0.93 if two else 0.67, 64: 0.57 if two else 0.3}[tile]
    return 4.0 + -(-tiles // (2 * cus if two else cus)) * (-(-k // 64) * unit + epi * {256: 7.0, 128: 4.0, 64: 1.5}[tile])


@pytest.mark.parametrize("what,sizes", [("gate", (391, 32, 9208)), ("gate", (43318, 21, 94)), ("gate", (100, 512, 1000)),
                                        ("dz", (37170, 138, 146)), ("dz", (1086, 283, 7189)), ("dz", (1229, 768, 30522)),
                                        ("last", (7, 192, 4864)), ("last", (11, 192, 3584)), ("last", (1, 4100, 2100))])
def test_plans_price_the_tiles_that_run(what, sizes):
    """Products whose kernels have two of the three tiles take the cheaper of those two."""
    if what == "gate":
        n, k, f = sizes
        got, tiles, args = _plan("gated_ffn", n, k, f)[0], (128, 256), (n, 2 * f, k, 1.5)
    elif what == "dz":
        n, k, v = sizes
        got, tiles, args = _plan("linear_cross_entropy", n, k, v, 1)[1], (64, 128), (n, v, k, 1.5)
    else:
        b, r, c = sizes
        side, length = (-(-min(r, c) // 64) * 64, -(-max(r, c) // 64) * 64)
        got, tiles, args = _plan("orthogonalize", b, r, c, 1)[3], (64, 128), (side, length * b, side)
    assert got == min(tiles, key=lambda t: _estimate(t, *args))


def test_fake_tensors_have_shapes():
    """Tensors without data go through the operators' checks to the shapes and types of their results."""
    from mihvd import _native
    from mihvd.ops import gated_ffn, linear_cross_entropy
    from mihvd.optim import orthogonalize
    from torch._subclasses.fake_tensor import FakeTensorMode

    if not _native.load_kernels():
        pytest.skip("no kernel library")
    with FakeTensorMode():
        def t(*s, dt=torch.bfloat16, **kw):
            return torch.empty(*s, dtype=dt, device="cuda:0", **kw)

        y = t(2, 5, dt=torch.long)
        for grad in (True, False):
            h, w, b = t(2, 5, 17, requires_grad=grad), t(33, 17, requires_grad=grad), t(33, dt=torch.float32)
            for red, shape in (("mean", ()), ("sum", ()), ("none", (2, 5))):
                out = linear_cross_entropy(h, w, y, b, reduction=red)
                assert out.shape == shape and out.dtype == torch.float32 and out.requires_grad == grad
            z = gated_ffn(h, t(12, 17), t(12, 17), t(17, 12), activation="gelu")
            assert z.shape == h.shape and z.dtype == h.dtype and z.requires_grad == grad
        x = t(3, 12, 17, dt=torch.float16)
        assert orthogonalize(x).shape == x.shape and orthogonalize(x).dtype == x.dtype


def test_muon_refuses_a_parameter_twice():
    from mihvd.optim import Muon

    p, q = torch.nn.Parameter(torch.ones(4, 3)), torch.nn.Parameter(torch.ones(4, 3))
    with pytest.raises(ValueError, match="twice"), pytest.warns(UserWarning, match="duplicate"):
        Muon([p, q, p])
    opt = Muon([q])
    with pytest.raises(ValueError, match="twice"), pytest.warns(UserWarning, match="duplicate"):
        opt.add_param_group(dict(params=[p, p]))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[p]))


def test_plan_refusals():
    from mihvd import _native

    if not _native.load_kernels():
        pytest.skip("no kernel library")
    for op, sizes in (("linear_cross_entropy", [0, 8, 8, 1]), ("linear_cross_entropy", [8, 8, 8]), ("gated_ffn", [8, 0, 8]),
                      ("gated_ffn", [8, 8, 8, 8]), ("orthogonalize", [0, 8, 8, 1]), ("orthogonalize", [1, 8, 8, 3]),
                      ("orthogonalize", [33, 8, 8, 1]), ("gated_ffn", [1 << 40, 8, 8]), ("softmax", [1, 2, 3])):
        with pytest.raises(ValueError, match="transformer_plan"):
            torch.ops.mihvd.transformer_plan(op, sizes)
