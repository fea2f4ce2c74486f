"""linear_cross_entropy, gated_ffn and Muon used together on the GPU, and the calls around them: captured and
replayed steps, streams, inference mode, two calls at once, many rows, differences, refusals."""
import json
import math
import os
import subprocess
import sys

import pytest
import torch

from test_transformer_gpu import BF, E32, FP, close, ffn_case, ffn_ref, gen, lce_case, lce_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _kernels():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from mihvd import _native

    _native.require_kernels()


class Stack:
    """Residual gated block, vocabulary loss, Muon on the three matrices and plain steps on the table: fp32
    weights under autocast."""

    def __init__(self, n=70, k=96, f=136, v=523):
        from mihvd.optim import Muon

        g = gen(5)
        self.x = torch.randn(n, k, generator=g).cuda()
        self.y = torch.randint(0, v, (n,), generator=g).cuda()
        self.y[::3] = -100
        self.w = [torch.nn.Parameter((torch.randn(s, generator=g) * by).cuda()) for s, by in
                  (((f, k), k ** -0.5), ((f, k), k ** -0.5), ((k, f), f ** -0.5))]
        self.table = torch.nn.Parameter((torch.randn(v, k, generator=g) * k ** -0.5).cuda())
        self.bias = torch.nn.Parameter(torch.zeros(v, device="cuda"))
        self.opt = Muon(self.w, lr=0.02, weight_decay=0.01)

    def loss(self):
        from mihvd.ops import gated_ffn, linear_cross_entropy

        with torch.autocast("cuda", torch.bfloat16):
            h = self.x + gated_ffn(self.x, *self.w)
            return linear_cross_entropy(h, self.table, self.y, self.bias)

    def step(self):
        for p in self.params():
            p.grad = None
        loss = self.loss()
        loss.backward()
        self.opt.step()
        with torch.no_grad():
            for p in (self.table, self.bias):
                p.sub_(p.grad, alpha=0.1)
        return loss.detach()

    def params(self):
        return [*self.w, self.table, self.bias]


def test_step_captured_and_replayed():
    a, b = Stack(), Stack()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # first steps off the default stream: the momenta exist before the capture
        b.step()
    torch.cuda.current_stream().wait_stream(side)
    a.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.step()
    for _ in range(4):
        want = a.step()
        torch.cuda.synchronize()
        graph.replay()
        junk = torch.randn(64, 64, device="cuda") @ torch.randn(64, 64, device="cuda")
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.isfinite(junk).all()
        for p, q in zip(a.params(), b.params()):
            assert torch.equal(p, q)


def test_first_muon_step_is_not_captured():
    s = Stack()
    for p in s.params():
        p.grad = torch.ones_like(p)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(graph):
            s.opt.step()
    torch.cuda.synchronize()
    s.opt.step()
    assert all(torch.isfinite(p).all() for p in s.params())


def test_two_graphs_share_nothing():
    """Two captured calls replayed in turn, each over its own inputs, keep their results."""
    from mihvd.ops import gated_ffn, linear_cross_entropy

    ins, outs, graphs, kept = [], [], [], []  # a graph reads its inputs where they were: they are kept
    for seed in (1, 2):
        h, w, y, b = lce_case(90, 72, 301, BF, torch.float32, seed)
        x, wg, wu, wd, _ = ffn_case(33, 72, 104, BF, seed)
        t = [q.cuda() for q in (h, w, y, b, x, wg, wu, wd)]

        def run(t=t):
            return linear_cross_entropy(*t[:4]), gated_ffn(*t[4:])

        want = run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run()
        kept.append(t)
        ins.append(want)
        outs.append(got)
        graphs.append(graph)
    for _ in range(3):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for want, got in zip(ins, outs):
            assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_capture_beside_a_live_eager_graph_is_refused():
    s = Stack()
    alive = s.loss()  # keeps the leaves' accumulators on the default stream
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(graph):
            s.loss().backward()
    torch.cuda.synchronize()
    del graph, alive
    for p in s.params():
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = s.loss()
        loss.backward()
    graph.replay()
    got = [p.grad.clone() for p in s.params()]
    t = Stack()
    t.loss().backward()
    assert all(torch.equal(p, q.grad) for p, q in zip(got, t.params()))


def test_other_streams_and_two_calls_at_once():
    from mihvd.ops import gated_ffn, linear_cross_entropy

    h, w, y, b = (q.cuda() for q in lce_case(200, 136, 1000, BF, torch.float32, 3))
    x, wg, wu, wd, dy = (q.cuda() for q in ffn_case(150, 136, 200, BF, 4))

    def both():
        lh, lw = h.detach().requires_grad_(), w.detach().requires_grad_()
        lx, lg = x.detach().requires_grad_(), wg.detach().requires_grad_()
        out = linear_cross_entropy(lh, lw, y, b)
        z = gated_ffn(lx, lg, wu, wd)
        return (out, z, *torch.autograd.grad(out, [lh, lw]), *torch.autograd.grad(z, [lx, lg], dy))

    want = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(both())
    torch.cuda.synchronize()
    for run in got[0] + got[1]:
        assert all(torch.equal(p, q) for p, q in zip(run, want))


def test_inference_mode_and_no_double_backward():
    from mihvd.ops import gated_ffn, linear_cross_entropy

    h, w, y, b = (q.cuda() for q in lce_case(20, 64, 99, BF, torch.float32, 6))
    x, wg, wu, wd, dy = (q.cuda() for q in ffn_case(20, 64, 72, BF, 6))
    with torch.inference_mode():
        a, z = linear_cross_entropy(h, w, y, b), gated_ffn(x, wg, wu, wd)
    lh, lx = h.detach().requires_grad_(), x.detach().requires_grad_()
    out, z2 = linear_cross_entropy(lh, w, y, b), gated_ffn(lx, wg, wu, wd)
    assert torch.equal(a, out) and torch.equal(z, z2) and not z.requires_grad
    for o, leaf in ((out, lh), (z2.sum(), lx)):
        d, = torch.autograd.grad(o, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated again"):
            d.float().sum().backward()


@pytest.mark.parametrize("n", [16384, 16385, 40000])
def test_many_rows_keep_their_order(n):
    """Rows on both sides of the count ahead: losses and gradients land in their own rows."""
    from mihvd.ops import linear_cross_entropy

    h, w, y, _ = lce_case(n, 16, 24, BF, None, seed=n, drop=0.7)
    y[-1] = 3
    gr = torch.rand(n, generator=gen(n), dtype=torch.float64).float()
    loss, ltol, dh, dw, _ = lce_ref(h, w, y, None, gr.double(), BF)
    leaves = [h.cuda().requires_grad_(), w.cuda().requires_grad_()]
    rows = linear_cross_entropy(*leaves, y.cuda(), reduction="none")
    close(rows, loss, ltol, "rows")
    gh, gw = torch.autograd.grad(rows, leaves, gr.cuda())
    close(gh, *dh, "dh")
    close(gw, *dw, "dw")
    assert (gh[(y == -100).cuda()] == 0).all()
    tot = linear_cross_entropy(*leaves, y.cuda(), reduction="sum")
    # fp32 sum of n terms: at most log2 steps in trees plus n / 4096 in a thread
    close(tot, loss.sum(), float((loss != 0).sum()) * ltol + (n / 4096 + 20) * E32 * float(loss.abs().sum()), "sum")


def test_gradients_against_differences():
    """Central differences of the kernels' own values along steps that the 16-bit type holds exactly. The
    differences' truncation is what the same differences show in 64 bits."""
    from mihvd.ops import gated_ffn, linear_cross_entropy

    g = gen(12)

    def grid(*s):  # multiples of 2^-4 within one: a step of 2^-6 stays within bf16's eight digits
        return torch.randint(-15, 16, s, generator=g).double() / 16

    n, k, v = 24, 40, 67
    h, w, y = grid(n, k).to(BF), (grid(v, k) / 4).to(BF), torch.randint(0, v, (n,), generator=g)
    one = torch.ones(n, dtype=torch.float64)
    leaves = [h.cuda().requires_grad_(), w.cuda().requires_grad_()]
    grads = torch.autograd.grad(linear_cross_entropy(*leaves, y.cuda(), reduction="sum"), leaves)
    for i, step in ((0, 2.0 ** -6), (1, 2.0 ** -8)):
        d = (torch.randint(0, 2, (h, w)[i].shape, generator=g) * 2 - 1).double() * step
        ends, ends64, tol = [], [], 0.0
        for sign in (1, -1):
            p = [h, w]
            p[i] = (p[i].double() + sign * d).to(BF)
            assert torch.equal(p[i].double(), (h, w)[i].double() + sign * d)
            ends.append(float(linear_cross_entropy(p[0].cuda(), p[1].cuda(), y.cuda(), reduction="sum").double()))
            loss, ltol, *_ = lce_ref(p[0], p[1], y, None, one, BF)
            ends64.append(float(loss.sum()))
            tol += n * ltol + n * E32 * float(loss.sum())
        _, _, *ref = lce_ref(h, w, y, None, one, BF)
        trunc = abs(ends64[0] - ends64[1] - 2 * float((ref[i][0] * d).sum()))
        tol += trunc + 2 * float((ref[i][1] * d.abs()).sum())
        assert abs(ends[0] - ends[1] - 2 * float((grads[i].double().cpu() * d).sum())) <= tol, i

    n, k, f = 12, 24, 40
    p = [grid(n, k).to(BF), (grid(f, k) / 4).to(BF), (grid(f, k) / 4).to(BF), (grid(k, f) / 4).to(BF)]
    dy = grid(n, k).to(BF)
    leaves = [t.cuda().requires_grad_() for t in p]
    grads = torch.autograd.grad(gated_ffn(*leaves), leaves, dy.cuda())
    ref = ffn_ref(*p, dy, "silu", BF)
    for i in range(4):
        d = (torch.randint(0, 2, p[i].shape, generator=g) * 2 - 1).double() * (2.0 ** -6 if i == 0 else 2.0 ** -8)
        ends, ends64, tol = [], [], 0.0
        for sign in (1, -1):
            q = list(p)
            q[i] = (p[i].double() + sign * d).to(BF)
            ends.append(float((gated_ffn(*(t.cuda() for t in q)).double().cpu() * dy.double()).sum()))
            yv, ye = ffn_ref(*q, dy, "silu", BF)[0]
            ends64.append(float((yv * dy.double()).sum()))
            tol += float((ye * dy.double().abs()).sum())
        trunc = abs(ends64[0] - ends64[1] - 2 * float((ref[1 + i][0] * d).sum()))
        tol += trunc + 2 * float((ref[1 + i][1] * d.abs()).sum())
        assert abs(ends[0] - ends[1] - 2 * float((grads[i].double().cpu() * d).sum())) <= tol, i


def test_operators_inside_and_outside_autocast():
    from mihvd.ops import gated_ffn, linear_cross_entropy

    x, wg, wu, wd, _ = (q.cuda() for q in ffn_case(6, 32, 40, FP, 8))
    h, w, y, b = (q.cuda() for q in lce_case(6, 32, 45, FP, torch.float32, 8))
    with torch.autocast("cuda", FP):
        assert torch.equal(gated_ffn(x.float(), wg.float(), wu.float(), wd.float()), gated_ffn(x, wg, wu, wd))
        assert torch.equal(linear_cross_entropy(h.float(), w.float(), y, b), linear_cross_entropy(h, w, y, b))
    with pytest.raises(TypeError, match="autocast"):
        gated_ffn(x.float(), wg, wu, wd)
    with pytest.raises(TypeError, match="autocast"):
        linear_cross_entropy(h.float(), w, y)
    with pytest.raises(TypeError, match="type"):
        gated_ffn(x, wg.bfloat16(), wu, wd)
    with pytest.raises(TypeError, match="bias"):
        linear_cross_entropy(h, w, y, b.double())
    with pytest.raises(ValueError, match="bias"):
        linear_cross_entropy(h, w, y, b[:-1])
    with pytest.raises(ValueError, match="GPU"):
        gated_ffn(x, wg.cpu(), wu, wd)


@pytest.mark.parametrize("ffn", ["geglu", "swiglu"])
def test_bert_step_with_all_three(ffn):
    """The BERT model with the gated block, the fused loss and Muon: its loss is the torch path's up to the
    rounding of logits to bf16, its gradients lie along the torch path's, and a step moves every parameter."""
    from mihvd.models.bert import BertConfig, BertForMaskedLM, muon_parameters, synthetic_mlm_batch
    from mihvd.optim import FusedAdam, Muon

    torch.manual_seed(0)
    c = BertConfig(vocab_size=301, hidden=64, layers=2, heads=2, ffn=96, max_len=32, dropout=0.0, ffn_impl=ffn,
                   loss_impl="fused")
    model = BertForMaskedLM(c).cuda()
    ids, labels = synthetic_mlm_batch(3, 31, 301, "cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    ids, labels = ids.clamp_max(300), labels.clamp_max(300)
    grads, losses = [], []
    for impl in ("fused", "torch"):
        model.c.loss_impl = impl
        model.zero_grad(set_to_none=True)
        with torch.autocast("cuda", torch.bfloat16):
            loss = model(ids, labels)
        loss.backward()
        losses.append(float(loss.detach()))
        grads.append([p.grad.detach().clone() for p in model.parameters()])
        del loss
    # a logit rounded to bf16 is off by 2^-8 of it; a row's loss is the difference of two such means
    assert abs(losses[0] - losses[1]) <= 2 * 2.0 ** -8 * 2.0 + 1e-3, losses
    a, b = (torch.cat([g.double().reshape(-1) for g in gs]) for gs in grads)
    # both are the same formula with bf16 rounding at every product (2^-8 each, under 32 of them on a path)
    assert float((a - b).norm()) <= 32 * 2.0 ** -8 * float(b.norm())
    matrices, others = muon_parameters(model)
    opts = [Muon(matrices, lr=0.02), FusedAdam(others, lr=1e-3)]
    before = [p.detach().clone() for p in model.parameters()]
    for p, g in zip(model.parameters(), grads[0]):
        p.grad = g
    for o in opts:
        o.step()
    moved = [not torch.equal(p, q) for p, q in zip(model.parameters(), before)]
    assert all(m or not g.any() for m, g in zip(moved, grads[0]))


def test_offsets_past_32_bits():
    """A block whose inner activations pass 2^31 elements (their gradients 2^32), and a vocabulary whose weight does:
    the last rows come out as a small call's formula says."""
    from mihvd.ops import gated_ffn, linear_cross_entropy

    n, k, f, tail = (1 << 20) + 77, 16, 2056, 40
    _, wg, wu, wd, _ = ffn_case(1, k, f, BF, 21)
    x = torch.randn(n, k, device="cuda").to(BF)
    dy = torch.randn(n, k, device="cuda").to(BF)
    xl = x.requires_grad_()
    y = gated_ffn(xl, wg.cuda(), wu.cuda(), wd.cuda())
    dx, = torch.autograd.grad(y, xl, dy)
    ref = ffn_ref(x[-tail:].detach().cpu(), wg, wu, wd, dy[-tail:].cpu(), "silu", BF)
    close(y[-tail:], *ref[0], "y")
    close(dx[-tail:], *ref[1], "dx")
    del y, dx, x, xl, dy

    v, k, n = (1 << 21) + 4099, 1032, 5
    w = torch.randn(v, k, device="cuda", dtype=torch.float32).mul_(k ** -0.5).to(BF)
    h = torch.randn(n, k, device="cuda").to(BF)
    labels = torch.tensor([v - 1, 0, v - 3, -100, 1 << 21], device="cuda")
    hl, wl = h.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(hl, wl, labels, reduction="sum")
    dh, dw = torch.autograd.grad(loss, [hl, wl])
    assert float(dh[3].abs().max()) == 0
    with torch.no_grad():
        z = torch.cat([h.double() @ w[i:i + (1 << 18)].double().t() for i in range(0, v, 1 << 18)], 1)
        p = torch.softmax(z, 1)
        keep = labels != -100
        zabs = 1032 * E32 * float((h.double().abs().sum(1) * w[-1000:].double().abs().max()).max())
        lse = torch.logsumexp(z, 1)
        want = (lse - z.gather(1, labels.clamp_min(0)[:, None]).squeeze(1))[keep]
        rel = 2 * zabs + 2 * 2.0 ** -18 + float(lse.abs().max()) * 2.0 ** -22
        assert abs(float(loss.double()) - float(want.sum())) <= 4 * rel + 16 * E32 * float(want.sum())
        dz = p.scatter_add(1, labels.clamp_min(0)[:, None], torch.full((n, 1), -1.0, device="cuda", dtype=torch.float64))
        dz *= keep[:, None]
        for part in (slice(v - 64, v), slice(1 << 21, (1 << 21) + 64), slice(0, 64)):
            d = dz[:, part]
            ref = d.t() @ h.double()
            err = (d.abs() * (2.0 ** -8 + 2.0 ** -21) + p[:, part] * keep[:, None] * rel + 2.0 ** -38).t() @ h.double().abs()
            close(dw[part], ref.cpu(), (err * 1.01 + ref.abs() * 2.0 ** -8).cpu(), "dw")


def test_stress_benchmark_with_all_three():
    """The stress benchmark's BERT step with the gated block, the fused loss and Muon, replayed from a graph."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, PYTHONPATH=root)
    for k in ("RANK", "WORLD_SIZE", "MASTER_PORT"):
        env.pop(k, None)
    p = subprocess.run([sys.executable, os.path.join(root, "benchmarks", "stress_models.py"), "--model", "bert-base",
                        "--steps", "3", "--warmup", "3", "--batch-size", "2", "--graph", "--bert-ffn", "swiglu", "--bert-loss",
                        "fused", "--optimizer", "muon"], env=env, capture_output=True, text=True, timeout=110)
    assert p.returncode == 0, p.stdout[-2000:] + p.stderr[-2000:]
    rec = json.loads(p.stdout.strip().splitlines()[-1])
    assert rec["config"]["optimizer"] == "muon" and math.isfinite(rec["config"]["final_loss"])
