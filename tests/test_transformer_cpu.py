"""The transformer-step operators without a GPU: refusals, the CPU forms of orthogonalize and Muon, the BERT
options, a two-rank Muon run, and a look at the built kernels' code."""
import copy
import json
import math
import os
import re
import shutil
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def ns64(x, steps=5, coef=(3.4445, -4.7750, 2.0315), eps=1e-7):
    a, b, c = coef
    z = x.double()
    z = z / (torch.linalg.vector_norm(z) + eps)
    for _ in range(steps):
        s = z @ z.t()
        z = a * z + (b * s + c * (s @ s)) @ z
    return z


@pytest.mark.parametrize("m,n", [(1, 1), (1, 5), (6, 1), (12, 7), (7, 12), (20, 20)])
def test_orthogonalize_cpu(m, n):
    from mihvd.optim import orthogonalize

    x = torch.randn(m, n, generator=torch.Generator().manual_seed(m * 31 + n))
    want = ns64(x)
    got = orthogonalize(x)
    # fp32 throughout: 64 roundings of 2^-24, an error growing at most fivefold a step relative to the values
    assert float((got.double() - want).norm()) <= 64 * 5 * 2.0 ** -24 * float(want.norm())
    assert orthogonalize(x.bfloat16()).dtype == torch.bfloat16
    # a stack sums in another order than one matrix: each lies within the bound above of the same value, so
    # by the triangle inequality the two lie within twice that bound of each other
    both = orthogonalize(torch.stack([x, 2 * x]))[0]
    assert float((both.double() - got.double()).norm()) <= 2 * 64 * 5 * 2.0 ** -24 * float(want.norm())


def test_orthogonalize_refusals():
    from mihvd.optim import orthogonalize

    x = torch.randn(4, 4)
    with pytest.raises(ValueError, match="matrix"):
        orthogonalize(x[0])
    with pytest.raises(TypeError, match="float32"):
        orthogonalize(x.double())
    with pytest.raises(ValueError, match="precision"):
        orthogonalize(x, precision="bf16")
    with pytest.raises(ValueError, match="steps"):
        orthogonalize(x, steps=-1)
    for bad in ((1.0, 2.0), (9.0, -5.0, 2.0), (1.0, float("nan"), 0.0)):
        with pytest.raises(ValueError, match="coefficients"):
            orthogonalize(x, coefficients=bad)
    assert orthogonalize(torch.zeros(0, 4)).shape == (0, 4) and orthogonalize(torch.zeros(2, 3, 0)).shape == (2, 3, 0)


def test_muon_refusals_and_cpu_steps():
    from mihvd.optim import Muon

    w = torch.nn.Parameter(torch.randn(6, 4, generator=torch.Generator().manual_seed(3)))
    for kw, word in ((dict(lr=-1.0), "lr"), (dict(momentum=1.0), "momentum"), (dict(scale="adam"), "scale"),
                     (dict(precision="fp8"), "precision"), (dict(ns_steps=101), "ns_steps"),
                     (dict(ns_coefficients=(1.0,)), "coefficients"), (dict(weight_decay=-0.1), "weight_decay")):
        with pytest.raises(ValueError, match=word):
            Muon([w], **kw)
    with pytest.raises(ValueError, match="two dimensions"):
        Muon([w, torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(TypeError, match="float64"):
        Muon([torch.nn.Parameter(torch.zeros(4, 4, dtype=torch.float64))])
    opt = Muon([w], lr=0.05, momentum=0.9, weight_decay=0.1, scale="rms")
    ref, mom = w.detach().double().clone(), torch.zeros(6, 4, dtype=torch.float64)
    for k in range(3):
        d = torch.randn(6, 4, generator=torch.Generator().manual_seed(10 + k))
        w.grad = d.clone()
        opt.step()
        mom = 0.9 * mom + d.double()
        ref = ref * (1 - 0.05 * 0.1) - 0.05 * 0.2 * math.sqrt(6) * ns64((d.double() + 0.9 * mom).t()).t()
    # the update is about 0.05 * 0.49 * 2 in norm a step, off by the bound of test_orthogonalize_cpu
    assert float((w.detach().double() - ref).norm()) <= 3 * (320 * 2.0 ** -24 * 0.1 + 2.0 ** -23 * float(ref.norm()))
    # a checkpoint's copy: load_state_dict itself keeps the tensors that it is given, as torch's optimizers do
    state = copy.deepcopy(opt.state_dict())
    w2 = torch.nn.Parameter(w.detach().clone())
    opt2 = Muon([w2], lr=0.05, momentum=0.9, weight_decay=0.1, scale="rms")
    opt2.load_state_dict(state)
    for p, o in ((w, opt), (w2, opt2)):
        p.grad = torch.ones(6, 4)
        o.step()
    assert torch.equal(w, w2)


def test_operator_refusals_cpu():
    from mihvd.ops import gated_ffn, linear_cross_entropy

    h, w, y = torch.randn(3, 8).bfloat16(), torch.randn(5, 8).bfloat16(), torch.zeros(3, dtype=torch.long)
    with pytest.raises(ValueError, match="GPU"):
        linear_cross_entropy(h, w, y)
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(h, w, y, reduction="max")
    with pytest.raises(ValueError, match="hidden"):
        linear_cross_entropy(h, w[:, :4], y)
    with pytest.raises(ValueError, match="labels"):
        linear_cross_entropy(h, w, y[:2])
    with pytest.raises(TypeError, match="int64"):
        linear_cross_entropy(h, w, y.int())
    g, d = torch.randn(6, 8).bfloat16(), torch.randn(8, 6).bfloat16()
    with pytest.raises(ValueError, match="GPU"):
        gated_ffn(h, g, g, d)
    with pytest.raises(ValueError, match="activation"):
        gated_ffn(h, g, g, d, activation="tanh")
    with pytest.raises(ValueError, match="w_down"):
        gated_ffn(h, g, g, g)
    with pytest.raises(ValueError, match="w_up"):
        gated_ffn(h, g, g[:5], d)


def test_bert_options_cpu():
    from mihvd.models.bert import BertConfig, BertForMaskedLM, flops_per_token, muon_parameters, synthetic_mlm_batch

    kw = dict(vocab_size=61, hidden=16, layers=2, heads=2, ffn=24, max_len=8, dropout=0.0)
    for bad in (dict(ffn_impl="glu"), dict(loss_impl="mse")):
        with pytest.raises(ValueError):
            BertForMaskedLM(BertConfig(**kw, **bad))
    g = torch.Generator().manual_seed(1)
    ids, labels = synthetic_mlm_batch(2, 8, 61, "cpu", generator=g, mask_prob=0.5)
    ids = ids.clamp_max(60)
    torch.manual_seed(0)
    m = BertForMaskedLM(BertConfig(**kw, ffn_impl="geglu", loss_impl="fused"))
    a = m(ids, labels)
    m.c.loss_impl = "torch"
    assert torch.equal(a, m(ids, labels))  # without a GPU both are the torch form
    a.backward()
    matrices, others = muon_parameters(m)
    assert len(matrices) == 2 * 5 and all(p.dim() == 2 and p.grad is not None for p in matrices)
    assert sum(p.numel() for p in matrices + others) == sum(p.numel() for p in m.parameters())
    x = torch.randn(3, 16)
    lay = m.layers[0]
    want = (torch.nn.functional.gelu(x @ lay.fc_gate.weight.t()) * (x @ lay.fc_up.weight.t())) @ lay.fc_down.weight.t()
    assert torch.allclose(lay._ffn(x), want, atol=1e-6)
    assert flops_per_token(BertConfig(ffn=2048, ffn_impl="swiglu"), 512) > flops_per_token(BertConfig(ffn=2048), 512)


@pytest.mark.slow
def test_muon_two_ranks_match_one(tmp_path):
    """Two gloo ranks on half the batch each end where one process on the whole batch ends."""
    worker = os.path.join(ROOT, "tests", "workers", "muon_worker.py")
    env = dict(os.environ, MIHVD_BACKEND="gloo", PYTHONPATH=ROOT, CUDA_VISIBLE_DEVICES="", HIP_VISIBLE_DEVICES="")
    for k in ("RANK", "WORLD_SIZE", "LOCAL_RANK", "LOCAL_WORLD_SIZE", "MASTER_PORT"):
        env.pop(k, None)
    flat = {}
    for n in (1, 2):
        out = str(tmp_path / ("w%d" % n))
        p = subprocess.run([sys.executable, "-m", "mihvd.runner", "-np", str(n), sys.executable, worker, out], env=env, cwd=ROOT,
                           capture_output=True, text=True, timeout=180)
        assert p.returncode == 0, p.stdout + p.stderr
        flat[n] = [torch.tensor(json.load(open("%s.%d.json" % (out, r)))) for r in range(n)]
    assert torch.equal(flat[2][0], flat[2][1])
    # the gradients differ by the rounding of a sum in two halves; Adam's first steps have slope lr / |g|
    assert float((flat[2][0] - flat[1][0]).abs().max()) <= 2e-4


def _regs(tok):
    m = re.match(r"([av])\[(\d+):(\d+)\]$", tok)
    if m:
        return {(m.group(1), i) for i in range(int(m.group(2)), int(m.group(3)) + 1)}
    m = re.match(r"([av])(\d+)$", tok)
    return {(m.group(1), int(m.group(2)))} if m else set()


def _early_uses(lines):
    """Instructions within 16 wait states behind an MFMA, along any path, that touch its result. `lines`: a
    kernel's (address, instruction, branch target or None)."""
    at = {a: i for i, (a, _, _) in enumerate(lines)}
    found = []
    for i, (_, s, _) in enumerate(lines):
        if not s.startswith("v_mfma"):
            continue
        acc = _regs(s.replace(",", " ").split()[1])
        stack, seen = [(i + 1, 0)], set()
        while stack:
            j, w = stack.pop()
            while j < len(lines) and w < 16 and (j, w) not in seen:
                seen.add((j, w))
                _, t, to = lines[j]
                p = t.replace(",", " ").split()
                if p[0] == "s_endpgm":
                    break
                if p[0] == "s_nop":
                    w += int(p[1]) + 1
                elif p[0].startswith("v_mfma"):
                    w += 1
                else:
                    if set().union(*[_regs(x) for x in p[1:]] or [set()]) & acc:
                        found.append((s, t, w))
                        break
                    w += 1
                    if to is not None and to in at:
                        stack.append((at[to], w))
                        if p[0] == "s_branch":
                            break
                j += 1
    return found


def test_products_leave_their_accumulators_alone(tmp_path):
    """The product kernels' MFMAs are asm blocks that accumulate in place: the compiler knows nothing of the
    matrix pipe's latency there, so no other instruction of theirs may touch an accumulator until the pipe
    is done (the kernels wait 16 states ahead of their epilogues). Read off the built library."""
    from mihvd import _build

    tool = "/opt/rocm/llvm/bin/llvm-objdump"
    if not os.path.exists(tool):
        pytest.skip("no llvm-objdump")
    if not os.path.exists(_build.KERNELS_SO):
        _build.build_kernels()
    names = ["linear_ce.hip.o", "linear_ce.hip.f16.o", "gated_ffn.hip.o", "gated_ffn.hip.f16.o", "newton_schulz.hip.o"]
    kernels = 0
    for name in names:
        src = os.path.join(_build.BUILD, name)
        obj = str(tmp_path / name)
        if not os.path.exists(src):
            pytest.skip("no object files beside the library")
        shutil.copy(src, obj)
        subprocess.run([tool, "--offloading", obj], cwd=tmp_path, capture_output=True, check=True)
        codes = [f for f in os.listdir(tmp_path) if f.startswith(name + ".") and "gfx950" in f]
        assert codes, os.listdir(tmp_path)
        for code in codes:
            text = subprocess.run([tool, "-d", "--no-show-raw-insn", str(tmp_path / code)], capture_output=True, text=True,
                                  check=True).stdout
            body, label = [], None
            for line in text.splitlines() + ["0 <end>:"]:
                head = re.match(r"^([0-9a-f]+) <(\S+)>:", line)
                if head:
                    if label and "gemm16_kernel" in label:
                        kernels += 1
                        assert not _early_uses(body), (name, label, _early_uses(body)[:3])
                    label, body, first = head.group(2), [], int(head.group(1), 16)
                    continue
                ins = re.match(r"^\s+(\S.*?)\s*//\s*([0-9A-Fa-f]+):", line)
                if ins:
                    to = re.search(r"<\S+?(?:\+0x([0-9a-f]+))?>\s*$", line)
                    is_branch = ins.group(1).startswith(("s_branch", "s_cbranch"))
                    target = first + int(to.group(1) or "0", 16) if to and is_branch else None
                    body.append((int(ins.group(2), 16), ins.group(1).strip(), target))
    assert kernels > 50, kernels
