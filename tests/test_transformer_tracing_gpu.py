"""The transformer-step operators under tracing on the GPU: what fake tensors say of their outputs is what the
kernels give, and whole-graph compilation (without a code generator) gives the eager results bit for bit."""
import pytest
import torch

from test_transformer_gpu import BF, FP, ffn_case, gen, lce_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _kernels():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from mihvd import _native

    _native.require_kernels()
    yield
    torch._dynamo.reset()


@pytest.mark.parametrize("dt", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("n,k,f", [(5, 17, 33), (70, 72, 104), (0, 16, 24)])
def test_fake_outputs_are_the_kernels(n, k, f, dt):
    ops = torch.ops.mihvd
    h, w, y, b = (t.cuda() for t in lce_case(max(n, 1), k, f, dt, torch.float32, n))
    h, y = h[:n], y[:n]
    checks = ("test_schema", "test_faketensor")
    for red in range(3):
        args = (h, w, y, b, -100, red)
        torch.library.opcheck(ops._linear_cross_entropy.default, args, test_utils=checks)
        loss, hc, meta, lse = ops._linear_cross_entropy(*args)
        for need in ((True, True, True), (False, True, False), (True, False, False)):
            torch.library.opcheck(ops._linear_cross_entropy_backward.default,
                                  (torch.ones_like(loss), hc, w, b, meta, lse, red, *need), test_utils=checks)
    x, wg, wu, wd, dy = (t.cuda()[:n] if i in (0, 4) else t.cuda() for i, t in enumerate(ffn_case(max(n, 1), k, f, dt, n)))
    torch.library.opcheck(ops._gated_ffn.default, (x, wg, wu, wd, 0), test_utils=checks)
    torch.library.opcheck(ops._gated_ffn_train.default, (x, wg, wu, wd, 1), test_utils=checks)
    mid = ops._gated_ffn_train(x, wg, wu, wd, 1)[1:]
    for need in ((True,) * 4, (False, False, True, False)):
        torch.library.opcheck(ops._gated_ffn_backward.default, (dy, x, wg, wu, wd, *mid, 1, *need), test_utils=checks)
    z = torch.randn(2, k, f, device="cuda").to(dt)
    torch.library.opcheck(ops.newton_schulz.default, (z, 5, 3.4445, -4.7750, 2.0315, 1e-7, False), test_utils=checks)


def head_and_block(x, wg, wu, wd, table, bias, y):
    from mihvd.ops import gated_ffn, linear_cross_entropy

    with torch.autocast("cuda", BF):
        h = x + gated_ffn(x, wg, wu, wd, activation="gelu")
        return linear_cross_entropy(h, table, y, bias)


@pytest.mark.parametrize("dynamic", [False, True])
def test_full_graph_compilation(dynamic):
    torch._dynamo.reset()
    fn = torch.compile(head_and_block, fullgraph=True, backend="aot_eager", dynamic=dynamic)
    for n in (40, 56):
        g = gen(n)
        shapes = ((n, 48), (72, 48), (72, 48), (48, 72), (99, 48), (99,))
        leaves = [(torch.randn(*s, generator=g) * 0.2).cuda().requires_grad_() for s in shapes]
        y = torch.randint(0, 99, (n,), generator=g).cuda()
        y[::5] = -100
        want = head_and_block(*leaves, y)
        ref = torch.autograd.grad(want, leaves)
        got = fn(*leaves, y)
        assert torch.equal(got, want)
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(got, leaves), ref))
        with torch.no_grad():
            assert torch.equal(fn(*leaves, y), want)


@pytest.mark.parametrize("ffn", ["gelu", "swiglu"])
def test_bert_full_graph(ffn):
    """The BERT model with the fused loss (and a gated block) compiles as one graph."""
    from mihvd.models.bert import BertConfig, BertForMaskedLM, synthetic_mlm_batch

    torch._dynamo.reset()
    torch.manual_seed(0)
    model = BertForMaskedLM(BertConfig(vocab_size=301, hidden=64, layers=2, heads=2, ffn=96, max_len=32, dropout=0.0,
                                       ffn_impl=ffn, loss_impl="fused")).cuda()
    ids, labels = synthetic_mlm_batch(3, 31, 301, "cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    ids, labels = ids.clamp_max(300), labels.clamp_max(300)
    step = torch.compile(model, fullgraph=True, backend="aot_eager")
    losses = []
    for call in (model, step):
        with torch.autocast("cuda", BF):
            loss = call(ids, labels)
        grads = torch.autograd.grad(loss, list(model.parameters()))
        losses.append((loss.detach(), grads))
    (a, ga), (b, gb) = losses
    # the same kernels on the same values, but for torch's own operators, which a trace may decompose: bf16 roundings
    assert abs(float(a) - float(b)) <= 2 * 2.0 ** -8 * 2.0
    flat = [torch.cat([t.double().reshape(-1) for t in gs]) for gs in (ga, gb)]
    assert float((flat[0] - flat[1]).norm()) <= 32 * 2.0 ** -8 * float(flat[0].norm())
