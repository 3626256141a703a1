"""The models on the operators of ops.train: the same tensors as their gradient sets, the same
results on a CPU as plain torch, on a GPU the operators, one by one and in data-parallel steps."""
import json
import os
import subprocess
import sys

import pytest
import torch
from torch.nn import functional as F

from stdml_collective_experimental_b200 import ops
from stdml_collective_experimental_b200.models import gradsets
from stdml_collective_experimental_b200.models.bert import Bert, bert_base, bert_large
from stdml_collective_experimental_b200.models.resnet import ResNet50

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
gpu = pytest.mark.gpu


def test_group_norm_resnet_has_the_tensors_of_its_set():
    with torch.device("meta"):
        sizes = sorted(p.numel() for p in ResNet50(norm="group").parameters())
        assert sizes == sorted(gradsets.gradset_sizes("resnet50"))
    with pytest.raises(ValueError, match="unknown norm"):
        ResNet50(norm="layer")


def test_gated_bert_keeps_about_its_parameters():
    with torch.device("meta"):
        for make, name in ((bert_base, "bert-base"), (bert_large, "bert-large")):
            plain, gated = (sum(p.numel() for p in make(**kw).parameters()) for kw in ({}, {"gated": True}))
            assert plain == sum(gradsets.gradset_sizes(name)) and abs(gated / plain - 1) < 0.002


def tiny_bert(**kw):
    torch.manual_seed(0)
    return Bert(2, 64, 4, 96, vocab=211, max_pos=32, dropout=0.0, gated=True, **kw)


def test_models_run_on_a_cpu():
    torch.manual_seed(0)
    model = ResNet50(num_classes=10, norm="group")
    y = model(torch.randn(2, 3, 32, 32))
    y.sum().backward()
    assert y.shape == (2, 10) and all(p.grad is not None for p in model.parameters())
    bert = tiny_bert()
    seq, pooled = bert(torch.randint(0, 211, (3, 9)))
    (bert.vocab_logits(seq).logsumexp(-1).sum() + pooled.sum()).backward()
    assert all(p.grad is not None for p in bert.parameters())


def relative(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@gpu
def test_group_norm_resnet_on_a_gpu_against_plain_torch():
    """f32 with TF32 off: the same network on a CPU in 64 bits.  Fifty layers of f32, each a few 2^-24 off and
    halving nothing: 2^-24 * 50 * 64 = 2e-4 bounds the outputs; gradients pass through them twice."""
    torch.manual_seed(0)
    model = ResNet50(num_classes=10, norm="group").eval()
    x = torch.randn(2, 3, 64, 64)
    ref = ResNet50(num_classes=10, norm="group").double()
    ref.load_state_dict({k: v.double() for k, v in model.state_dict().items()})
    want = ref(x.double())
    want.square().sum().backward()
    tf32 = torch.backends.cudnn.allow_tf32
    torch.backends.cudnn.allow_tf32 = False
    try:
        for layout in (torch.contiguous_format, torch.channels_last):
            mine = model.cuda().to(memory_format=layout)
            mine.zero_grad()
            y = mine(x.cuda().to(memory_format=layout))
            y.square().sum().backward()
            assert relative(y.cpu(), want) < 2e-4
            got = torch.cat([p.grad.cpu().flatten() for p in mine.parameters()])
            assert relative(got, torch.cat([p.grad.flatten() for p in ref.parameters()])) < 4e-4
    finally:
        torch.backends.cudnn.allow_tf32 = tf32


@gpu
def test_gated_bert_on_a_gpu_against_plain_torch():
    bert = tiny_bert()
    ids = torch.randint(0, 211, (3, 9), generator=torch.Generator().manual_seed(1))
    ref = tiny_bert().double()
    seq, pooled = ref(ids)
    (seq.square().sum() + pooled.sum()).backward()
    mine = bert.cuda()
    s, p = mine(ids.cuda())
    (s.square().sum() + p.sum()).backward()
    assert relative(s.cpu(), seq) < 2e-5
    got = torch.cat([q.grad.cpu().flatten() for q in mine.parameters()])
    assert relative(got, torch.cat([q.grad.flatten() for q in ref.parameters()])) < 1e-4
    # under autocast the block takes 16-bit operands, as nn.Linear does there: some ten roundings of 2^-9 on the way
    with torch.autocast("cuda", dtype=torch.bfloat16):
        block = mine.layers[0].up
        x = torch.randn(5, 64, device="cuda")
        h = block(x)
        assert h.dtype == torch.bfloat16
        s16, _ = mine(ids.cuda())
    assert relative(s16.float().cpu(), seq) < 10 * 2.0 ** -8


@gpu
def test_data_parallel_steps_of_students():
    """A session of one rank: gradients land in the symmetric heap's views, the same as without it."""
    from stdml_collective_experimental_b200 import DeviceSession
    from stdml_collective_experimental_b200.parallel.ddp import DataParallel
    ids = torch.randint(0, 211, (4, 12), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    top, index = torch.topk(torch.randn(4, 12, 211, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)), 9)
    labels = ids.masked_fill(ids % 3 == 0, -100)

    def loss_of(model, bert):
        return ops.distill_loss(bert.vocab_logits(model(ids)[0]), top, index, labels, temperature=2.0)

    plain = tiny_bert().cuda()
    loss_of(plain, plain).backward()
    want = [p.grad.clone() if p.grad is not None else torch.zeros_like(p) for p in plain.parameters()]
    with DeviceSession.from_env(heap_bytes=64 << 20, rank=0, world=1, device=0) as sess:
        bert = tiny_bert().cuda()
        model = DataParallel(bert, sess, buckets=3)
        for _ in range(2):
            model.zero_grad()
            loss_of(model, bert).backward()
        torch.cuda.synchronize()
        sess.check()
        ops.check()
        for p, w in zip(bert.parameters(), want):
            assert torch.allclose(p.grad, w, rtol=1e-5, atol=1e-6)
        with model.no_sync():  # accumulates
            loss_of(model, bert).backward()
        torch.cuda.synchronize()
        for p, w in zip(bert.parameters(), want):
            assert torch.allclose(p.grad, 2 * w, rtol=1e-5, atol=1e-6)
        model.close()


@gpu
@pytest.mark.parametrize("args", [
    ["--model", "resnet50", "--batch", "4", "--norm", "group", "--teacher", "5"],
    ["--model", "bert-base", "--batch", "2", "--seq", "37", "--ffn", "gated", "--teacher", "16"],
])
def test_benchmark_command(args):
    env = dict(os.environ, RANK="0", WORLD_SIZE="1", LOCAL_RANK="0")
    res = subprocess.run([sys.executable, "-m", "stdml_collective_experimental_b200.benchmarks.resnet50_dp", "--mode", "ours",
                          "--steps", "2", "--warmup", "1", *args], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
    line = json.loads(res.stdout.strip().splitlines()[-1])
    assert line["mode"] == "ours" and line["loss"] == line["loss"] and line["teacher"] == int(args[-1])


def test_plain_forms_agree_on_a_cpu():
    """What the modules compute off a GPU is what the operators are defined as."""
    bert = tiny_bert()
    block, x = bert.layers[0].up, torch.randn(4, 64)
    want = F.gelu(x @ block.gate.weight.t() + block.gate.bias) * (x @ block.up.weight.t() + block.up.bias)
    assert torch.allclose(block(x), want, atol=1e-6)
