"""linear_cross_entropy, gated_ffn, orthogonalize and Muon at the ends of their ranges on the GPU: masks of any
size over whole runs of words, sizes that every tile and piece serves, row counts past the launch limits, forward-mode
derivatives, 16-bit parameters over many steps. Compared with the formulas in 64 bits (computed on the GPU in
elementary operations where they are large)."""
import math

import pytest
import torch

from test_transformer_gpu import BF, E32, EXP, FP, close, floor_of, gen, half, lce_case, lce_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _kernels():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from mihvd import _native

    _native.require_kernels()


def lce_ref_gpu(h, w, y, b, grow, dt):
    """lce_ref with its sums on the GPU (sizes that take a CPU too long)."""
    loss, ltol, *rest = lce_ref(h.cuda(), w.cuda(), y.cuda(), None if b is None else b.cuda(), grow.cuda(), dt)
    return (loss.cpu(), ltol, *[tuple(t.cpu() if torch.is_tensor(t) else t for t in pair) for pair in rest])


# Sizes whose logits run in 64, 128 and 256 wide tiles: strips of 32, 64 and 128 words to a wave.
STRIPS = [(60, 64, 1111), (300, 100, 20000), (700, 136, 20011)]


@pytest.mark.parametrize("low", [-1e10, -1e30, torch.finfo(BF).min, torch.finfo(torch.float32).min, -math.inf],
                         ids=["1e10", "1e30", "bf16min", "fp32min", "inf"])
@pytest.mark.parametrize("n,k,v", STRIPS)
def test_lce_runs_of_masked_words(n, k, v, low):
    """Runs of words masked by one large value, across whole strips and tiles and at the vocabulary's end: what
    the formula gives over the words that are left; the masked words get exact zeros."""
    from mihvd.ops import linear_cross_entropy

    dt = BF if n != 300 else FP
    h, w, y, b = lce_case(n, k, v, dt, torch.float32, seed=n)
    off = torch.zeros(v, dtype=torch.bool)
    off[v // 4:v // 4 + 600] = True
    off[-300:] = True
    left = (~off).nonzero().squeeze(1)
    y = torch.where((y >= 0) & off[y.clamp(min=0)], left[y.clamp(min=0) % len(left)], y)
    cnt = int((y != -100).sum())
    scale = 64.0 if dt == FP else 1.0
    place = torch.cumsum(~off, 0) - 1  # a word's place among those that are left
    small = torch.where(y >= 0, place[y.clamp(min=0)], y)
    grow = torch.full((n,), scale / cnt, dtype=torch.float64)
    loss, ltol, dh, dw, db = lce_ref_gpu(h, w[left], small, b[left], grow, dt)
    b[off] = low
    bias = b.to(dt) if low == torch.finfo(BF).min and dt == BF else b
    if bias.dtype == dt:
        loss, ltol, dh, dw, db = lce_ref_gpu(h, w[left], small, bias[left], grow, dt)
    leaves = [t.cuda().requires_grad_() for t in (h, w, bias)]
    out = linear_cross_entropy(leaves[0], leaves[1], y.cuda(), leaves[2])
    close(out, loss.sum() / cnt, ltol + n * E32 * float(loss.abs().max()), "loss")
    gh, gw, gb = torch.autograd.grad(out, leaves, torch.tensor(scale, device="cuda"))
    close(gh, *dh, "dh")
    close(gw.cpu()[left], *dw, "dw")
    close(gb.cpu()[left], *db, "db")
    assert (gw.cpu()[off] == 0).all() and (gb.cpu()[off] == 0).all()


@pytest.mark.parametrize("low", [-1e10, -1e30, torch.finfo(torch.float32).min, 1e30], ids=["m1e10", "m1e30", "fp32min", "p1e30"])
@pytest.mark.parametrize("n,k,v", STRIPS)
def test_lce_all_words_alike(n, k, v, low):
    """Every word's bias is one value so large that the logits vanish beside it in 32 bits: the softmax is
    uniform, the loss log v, and the gradients are those of a uniform softmax."""
    from mihvd.ops import linear_cross_entropy

    h, w, y, _ = lce_case(n, k, v, BF, None, seed=n + 1)
    assert float((h.double() @ w.double().t()).abs().max()) < abs(low) * 2.0 ** -26
    keep = y != -100
    cnt = int(keep.sum())
    leaves = [h.cuda().requires_grad_(), w.cuda().requires_grad_()]
    b = torch.full((v,), low, device="cuda")
    out = linear_cross_entropy(leaves[0], leaves[1], y.cuda(), b)
    rel = 2 * EXP + math.log(v) * 2.0 ** -22
    close(out, torch.tensor(math.log(v), dtype=torch.float64), rel + 2 * n * E32 * math.log(v), "loss")
    gh, gw = torch.autograd.grad(out, leaves)
    p = torch.full((n, v), 1.0 / v, dtype=torch.float64)
    dz = p.clone()
    dz[torch.arange(n)[keep], y[keep]] -= 1.0
    g = (keep / cnt)[:, None]
    err = g * (dz.abs() * (2.0 ** -8 + 2.0 ** -21) + p * rel)
    dz = dz * g
    acc = dz.abs() + err
    want = dz @ w.double()
    close(gh, want, (err + acc * v * E32) @ w.double().abs() + want.abs() * 2.0 ** -8, "dh")
    want = dz.t() @ h.double()
    close(gw, want, (err + acc * n * E32).t() @ h.double().abs() + want.abs() * 2.0 ** -8, "dw")


def test_lce_rows_past_a_launch():
    """More rows than one launch has waves for (2^26 and some), in a pattern that repeats every 1024: every
    row's loss and gradient is its pattern's."""
    from mihvd.ops import linear_cross_entropy

    k, v, n, per = 8, 24, (1 << 26) + 37, 1024
    h, w, y, _ = lce_case(per, k, v, BF, None, seed=31)
    grow = torch.rand(per, generator=gen(32), dtype=torch.float64).float().double()
    loss, ltol, dh, _, _ = lce_ref(h, w, y, None, grow, BF)

    def pattern(t):
        return t.cuda().repeat(-(-n // per), *([1] * (t.dim() - 1)))[:n]

    hl = pattern(h).requires_grad_()
    rows = linear_cross_entropy(hl, w.cuda(), pattern(y), reduction="none")
    gh, = torch.autograd.grad(rows, hl, pattern(grow.float()))
    close(rows[:per], loss, ltol, "rows")
    close(gh[:per], *dh, "dh")
    for t in (rows.detach(), gh):
        whole = t[:n // per * per].view(-1, *t[:per].shape)
        assert (whole == whole[:1]).all() and torch.equal(t[n // per * per:], t[:n % per])
    del hl, rows, gh, t, whole
    torch.cuda.empty_cache()


def test_lce_hidden_gradient_past_a_launch():
    """A hidden gradient of more than 2^34 elements (one row's vector, expanded): rows of one label are alike to
    the last, ignored ones zero."""
    from mihvd.ops import linear_cross_entropy

    k, v, n = 4104, 16, (1 << 22) + 5
    h, w, _, _ = lce_case(1, k, v, BF, None, seed=33, drop=0.0)
    y = torch.arange(n) % 5
    y[y == 4] = -100
    hl = h.cuda().expand(n, k).detach().requires_grad_()
    loss = linear_cross_entropy(hl, w.cuda(), y.cuda(), reduction="sum")
    gh, = torch.autograd.grad(loss, hl)
    _, _, dh, _, _ = lce_ref(h.expand(5, k), w, y[:5], None, torch.ones(5, dtype=torch.float64), BF)
    close(gh[:5], *dh, "dh")
    for at in (n // 5 // 2 * 5, n - n % 5 - 50000):
        part = gh[at:at + 50000].view(-1, 5, k)
        assert (part == gh[:5]).all(), at
    assert torch.equal(gh[-(n % 5):], gh[:n % 5])
    del hl, loss, gh, part
    torch.cuda.empty_cache()


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("grad", [True, False], ids=["grad", "no_grad"])
def test_forward_mode_is_refused(which, grad):
    """A tangent on any input raises, with reverse mode on or off: it is never dropped for a zero derivative."""
    import torch.autograd.forward_ad as fwd

    from mihvd.ops import gated_ffn, linear_cross_entropy
    from test_transformer_gpu import ffn_case

    block = [t.cuda() for t in ffn_case(5, 16, 24, BF, 1)[:4]]
    h, w, y, b = (t.cuda() for t in lce_case(6, 16, 30, BF, torch.float32, 2))
    head = [h, w, b]
    with torch.set_grad_enabled(grad), fwd.dual_level():
        args = [fwd.make_dual(t, torch.ones_like(t)) if i == which else t for i, t in enumerate(block)]
        with pytest.raises(NotImplementedError, match="forward-mode"):
            gated_ffn(*args)
        if which < 3:
            args = [fwd.make_dual(t, torch.ones_like(t)) if i == which else t for i, t in enumerate(head)]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                linear_cross_entropy(args[0], args[1], y, args[2])
    if which < 1:
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(lambda t: gated_ffn(t, *block[1:]), (block[0],), (block[0],))
    assert torch.isfinite(gated_ffn(*block)).all()


def test_float64_is_not_cast_by_autocast():
    """Autocast leaves doubles alone, and so do the operators: they refuse them as they do without it."""
    from mihvd.ops import gated_ffn, linear_cross_entropy
    from test_transformer_gpu import ffn_case

    block = [t.cuda() for t in ffn_case(5, 16, 24, BF, 1)[:4]]
    h, w, y, b = (t.cuda() for t in lce_case(6, 16, 30, BF, torch.float32, 2))
    with torch.autocast("cuda", BF):
        for i in range(4):
            with pytest.raises(TypeError, match="bfloat16 or float16|type of the first"):
                gated_ffn(*[t.double() if i == j else t.float() for j, t in enumerate(block)])
        for i in range(2):
            with pytest.raises(TypeError, match="bfloat16 or float16|type of the first"):
                linear_cross_entropy(*[t.double() if i == j else t.float() for j, t in enumerate((h, w))], y)
        with pytest.raises(TypeError, match="bias"):
            linear_cross_entropy(h, w, y, b.double())


@pytest.mark.parametrize("dt", [BF, FP], ids=["bf16", "fp16"])
def test_muon_momentum_of_16_bit_parameters(dt):
    from test_transformer_ranges_cpu import muon_drift

    muon_drift(dt, "cuda")


def test_newton_schulz_coefficients_out_of_range():
    """Coefficients whose steps can pass what fp16 planes hold are refused before anything is written; those
    that stay within are computed, close to the bound too (a matrix of rank one starts at singular value one)."""
    from mihvd.optim import Muon, orthogonalize
    from test_transformer_gpu import ns64, ns_tol

    x = (torch.randn(20, 1, generator=gen(41)) @ torch.randn(1, 30, generator=gen(42))).cuda()
    for steps, coef in ((3, (4.0, -2.0, 1.0)), (3, (3.0, 0.0, 0.0)), (5, (2.0, 0.5, 0.0)), (2, (1.5, 1.0, 1.0))):
        with pytest.raises(ValueError, match="coefficients"):
            orthogonalize(x, steps=steps, coefficients=coef)
        p = torch.nn.Parameter(x.clone())
        p.grad = x.clone()
        opt = Muon([p], ns_steps=steps, ns_coefficients=coef)
        with pytest.raises(ValueError, match="coefficients"):
            opt.step()
        assert torch.equal(p, x)
    for steps, coef in ((2, (3.5, 0.0, 0.0)), (1, (10.0, -1.0, 4.0)), (5, (1.5, -0.5, 0.0)), (2, (1.2, 0.5, 0.2))):
        for dt in (torch.float32, FP):
            got = orthogonalize(x.to(dt), steps=steps, coefficients=coef).double().cpu()
            want = ns64(x.to(dt).cpu(), steps, coef)
            # |f'(s)| s <= 5 |f(s)| at the one singular value; what rounding puts beside it grows by at most 12
            tol = ns_tol(want, dt, dt == torch.float32)
            assert torch.linalg.vector_norm(got - want) <= tol, (steps, coef)


@pytest.mark.parametrize("dt", [torch.float32, BF], ids=["fp32", "bf16"])
def test_muon_step_counts_as_a_change(dt):
    """A graph that saved a weight before the step cannot be run backward with the weight after it, on the fused
    path and the other."""
    from mihvd.optim import Muon

    w = torch.nn.Parameter(torch.randn(16, 24, generator=gen(51)).cuda().to(dt))
    x = torch.randn(5, 24, generator=gen(52)).cuda().to(dt).requires_grad_()
    w.grad = torch.ones_like(w)
    opt = Muon([w], lr=0.1)
    y = (x @ w.t()).sum()
    before = w._version
    opt.step()
    m = opt.state[w]["momentum_buffer"]
    assert w._version > before and m._version > 0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    (x @ w.t()).sum().backward()
    wd = w.detach().double()
    # a sum of 16 weights, in fp32 (and rounded to bf16)
    tol = (16 * E32 + (half(dt) if dt == BF else 0)) * wd.abs().sum(0)
    close(x.grad, wd.sum(0).expand(5, 24).cpu(), tol.expand(5, 24).cpu(), "x.grad")
    with torch.inference_mode():
        opt.step()


@pytest.mark.parametrize("by,eps", [(2.0 ** 100, 1e-7), (2.0 ** 120, 1e-7), (2.0 ** -90, 0.0)])
@pytest.mark.parametrize("dt", [torch.float32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("m,n", [(70, 33), (20, 300)])
def test_orthogonalize_far_norms(m, n, dt, by, eps):
    """Values whose squares leave fp32's range have the result of their moderate multiple; a Muon step takes
    such gradients."""
    from mihvd.optim import Muon, orthogonalize
    from test_transformer_gpu import ns64, ns_tol

    x = torch.randn(2, m, n, generator=gen(61)).to(dt)
    got = orthogonalize((x * by).cuda(), eps=eps).double().cpu()
    for i in range(2):
        want = ns64(x[i], eps=0.0)
        assert torch.linalg.vector_norm(got[i] - want) <= ns_tol(want, dt, dt == torch.float32), i
    w = torch.nn.Parameter(torch.zeros(m, n, device="cuda", dtype=dt))
    w.grad = (x[0] * by).cuda()
    Muon([w], lr=1.0, momentum=0.5, eps=eps).step()
    want = ns64(x[0], eps=0.0) * math.sqrt(max(1.0, m / n))
    assert torch.linalg.vector_norm(w.detach().double().cpu() + want) <= 1.01 * ns_tol(want, dt, True)


def test_row_weights_and_masks_captured():
    """Per-row losses with weighted gradients and a masked vocabulary, captured once and replayed over new labels,
    weights and masks in the same tensors."""
    from mihvd.ops import linear_cross_entropy

    n, k, v = 90, 72, 700
    h, w, y, b = (t.cuda() for t in lce_case(n, k, v, BF, torch.float32, 71))
    gr = torch.rand(n, generator=gen(72)).cuda()

    def run():
        leaves = [t.detach().requires_grad_() for t in (h, w, b)]
        rows = linear_cross_entropy(leaves[0], leaves[1], y, leaves[2], reduction="none")
        return (rows.detach(), *torch.autograd.grad(rows, leaves, gr))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in range(4):
        g = gen(80 + seed)
        off = torch.zeros(v, dtype=torch.bool)
        off[100 * seed:100 * seed + 300] = True
        new = torch.randint(0, v, (n,), generator=g)
        new[off[new]] = -100
        if seed == 3:
            new.fill_(-100)  # nothing labelled
        y.copy_(new)
        gr.copy_(torch.randn(n, generator=g))
        b.copy_(torch.where(off, torch.tensor(-1e30), torch.randn(v, generator=g)))
        want = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want)), seed
        assert all(torch.isfinite(p).all() for p in want)


@pytest.mark.parametrize("dt", [BF, torch.float32], ids=["bf16", "fp32"])
def test_muon_captured(dt):
    """Steps of 16-bit parameters and of fp32 ones, channels_last among them, replayed from a graph."""
    from mihvd.optim import Muon

    def make():
        g = gen(91)
        ps = [torch.nn.Parameter(torch.randn(*s, generator=g).cuda().to(dt)) for s in ((24, 40), (40, 24), (16, 8, 3, 3))]
        ps[2].data = ps[2].data.to(memory_format=torch.channels_last)
        for p in ps:
            p.grad = torch.empty_like(p)
        return ps, Muon(ps, lr=0.05, weight_decay=0.1)

    (a, oa), (c, oc) = make(), make()

    def grads(seed):
        g = gen(seed)
        for p, q in zip(a, c):
            d = torch.randn(*p.shape, generator=g).cuda()
            p.grad.copy_(d)
            q.grad.copy_(d)

    grads(1)
    oa.step()
    oc.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oc.step()
    for seed in range(2, 6):
        grads(seed)
        oa.step()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(a, c):
            assert torch.equal(p, q) and torch.equal(oa.state[p]["momentum_buffer"], oc.state[q]["momentum_buffer"])


def test_threads_on_their_own_streams():
    """Two threads call the operators at once, each on a stream of its own."""
    import threading

    from mihvd.ops import gated_ffn, linear_cross_entropy
    from mihvd.optim import orthogonalize
    from test_transformer_gpu import ffn_case

    def work(seed):
        h, w, y, b = (t.cuda() for t in lce_case(150, 64, 900, BF, torch.float32, seed))
        x, wg, wu, wd, dy = (t.cuda() for t in ffn_case(40 + seed, 64, 200, BF, seed))
        lh, lx = h.requires_grad_(), x.requires_grad_()
        loss, z = linear_cross_entropy(lh, w, y, b), gated_ffn(lx, wg, wu, wd)
        return (loss.detach(), z.detach(), *torch.autograd.grad(loss, lh), *torch.autograd.grad(z, lx, dy),
                orthogonalize(w.float()[:100]))

    want = [work(s) for s in (1, 2)]
    torch.cuda.synchronize()
    bad = []

    def loop(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(5):
                got = work(i + 1)
                st.synchronize()
                if not all(torch.equal(p, q) for p, q in zip(got, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_capture_beside_an_eager_graph_of_a_side_stream():
    """The way out that the refusal names: an eager step run on a side stream may stay alive (as its loss does after
    a warm-up loop) while the next one is captured."""
    from test_transformer_steps_gpu import Stack

    s = Stack()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = s.loss()
        alive.backward()
    torch.cuda.current_stream().wait_stream(side)
    want = [p.grad.clone() for p in s.params()]
    for p in s.params():
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = s.loss()
        loss.backward()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, alive) and all(torch.equal(p.grad, q) for p, q in zip(s.params(), want))
