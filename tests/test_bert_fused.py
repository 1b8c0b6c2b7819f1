"""BERT with the fused layer norm, the fused masked-token loss and a teacher:
the operators together, as models/bert.py and benchmarks/bert_benchmark.py use
them."""
import os
import subprocess
import sys

import pytest
import torch

from dear_pytorch_amd import models
from dear_pytorch_amd.ops.fused_ln import FusedLayerNorm
from utils_dist import run_dist

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
VOCAB = 1000


def small(fused, hidden=48, layers=2):
    torch.manual_seed(0)
    return models.BertForPreTraining(models.BertConfig(
        vocab_size=VOCAB, hidden_size=hidden, num_hidden_layers=layers,
        num_attention_heads=4, intermediate_size=2 * hidden,
        max_position_embeddings=32, hidden_dropout_prob=0.0,
        attention_probs_dropout_prob=0.0, fused_ln=fused))


def batch(dev, B=4, S=17, seed=1, labelled=0.3):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, VOCAB, (B, S), generator=g)
    mlm = torch.where(torch.rand(B, S, generator=g) < labelled,
                      torch.randint(0, VOCAB, (B, S), generator=g), -1)
    mlm[0, 0] = 5
    nsp = torch.randint(0, 2, (B,), generator=g)
    mask = torch.ones(B, S, dtype=torch.long)
    mask[1, 11:] = 0                       # a padded sequence
    mlm[1, 11:] = -1
    return [t.to(dev) for t in (ids, torch.zeros_like(ids), mask, mlm, nsp)]


def step(model, crit, b, answers=None):
    model.zero_grad()
    scores, seq = model(*b[:3])
    loss = crit(scores, seq, b[3], b[4], *([] if answers is None
                                           else [answers]))
    loss.backward()
    return loss.detach(), {n: p.grad.clone()
                           for n, p in model.named_parameters()}


def off(a, ref):
    """Relative distance of all gradients together, in the 2-norm."""
    num = sum((a[n].double().cpu() - ref[n].cpu()).square().sum()
              for n in ref)
    return (num / sum(g.square().sum() for g in ref.values())).sqrt().item()


def test_fused_model_takes_the_plain_state_and_gives_its_numbers():
    plain, fused = small(False), small(True)
    fused.load_state_dict(plain.state_dict())
    assert sum(isinstance(m, FusedLayerNorm) for m in fused.modules()) == 6
    b = batch("cpu")
    crit = models.BertPretrainingCriterion(VOCAB)
    a, ga = step(plain, crit, b)
    c, gc = step(fused, crit, b)
    # float32 on the CPU: the same operations in the same order
    assert torch.equal(a, c)
    assert all(torch.equal(ga[n], gc[n]) for n in ga)


def test_fused_criterion_is_the_plain_one():
    model, b = small(False).double(), batch("cpu")
    a, ga = step(model, models.BertPretrainingCriterion(VOCAB), b)
    c, gc = step(model, models.BertPretrainingCriterion(VOCAB, fused=True), b)
    assert abs(a - c) < 1e-13 * a and off(ga, gc) < 1e-12
    none = torch.full_like(b[3], -1)       # no label: NaN from both
    for fused in (False, True):
        crit = models.BertPretrainingCriterion(VOCAB, fused=fused)
        with torch.no_grad():
            assert torch.isnan(crit(*model(*b[:3]), none, b[4]))


def test_distillation_criterion_follows_its_formula():
    model, b = small(False).double(), batch("cpu")
    teacher = small(False, hidden=64).double()
    crit = models.BertDistillationCriterion(VOCAB, top=VOCAB // 10,
                                            temperature=2.0, weight=0.25)
    said = crit.answers(teacher(*b[:3])[0], b[3])
    assert said.top_ids.shape == (4, 17, 100)
    assert not said.top_logprobs.requires_grad
    assert (said.top_ids >= 0).all(-1).equal(b[3] != -1)
    loss, grads = step(model, crit, b, said)
    model.zero_grad()
    scores, seq = model(*b[:3])
    plain = models.BertPretrainingCriterion(VOCAB)
    mlm = plain.masked_token_loss(scores, b[3])
    nsp = plain(scores, seq, b[3], b[4]) - mlm
    keep = b[3] != -1
    s = torch.log_softmax(scores[keep] / 2.0, -1)
    t = torch.log_softmax(teacher(*b[:3])[0][keep] / 2.0, -1).detach()
    ids = t.topk(100, -1)[1]
    named = torch.zeros_like(s, dtype=torch.bool).scatter(1, ids, True)
    bucket = lambda l: torch.cat([
        l.gather(1, ids), l.masked_fill(named, -torch.inf)
        .logsumexp(-1, keepdim=True)], -1)
    kl = (bucket(t).exp() * (bucket(t) - bucket(s))).sum(-1).mean() * 4.0
    want = 0.75 * mlm + 0.25 * kl + nsp
    want.backward()
    assert abs(loss - want) < 1e-12 * want
    assert off(grads, {n: p.grad for n, p in model.named_parameters()}) < 1e-11
    for bad in (dict(weight=1.5), dict(top=0), dict(top=129),
                dict(top=VOCAB + 1)):
        with pytest.raises(ValueError):
            models.BertDistillationCriterion(VOCAB, **bad)


def _rank_fused(rank, world):
    import dear_pytorch_amd as dear
    dear.init(backend="gloo")
    model = small(True)
    crit = models.BertDistillationCriterion(VOCAB, top=8)
    teacher = small(True, hidden=64).eval()
    opt = dear.DistributedOptimizer(
        torch.optim.SGD(model.parameters(), lr=0.1), model=model)
    for i in range(3):
        b = batch("cpu", seed=2 * i + rank, labelled=1.0)
        b[2].fill_(1)
        b[3][1, 11:] = 7
        with torch.no_grad():
            said = crit.answers(teacher(*b[:3])[0], b[3])
        opt.zero_grad()
        crit(*model(*b[:3]), b[3], b[4], said).backward()
        opt.step()
    opt.synchronize()
    out = {n: p.detach().clone().numpy() for n, p in model.named_parameters()}
    dear.shutdown()
    return out


def test_data_parallel_step_is_the_whole_batch_step():
    a, b = run_dist(_rank_fused, world_size=2)
    model = small(True)
    crit = models.BertDistillationCriterion(VOCAB, top=8)
    teacher = small(True, hidden=64).eval()
    opt = torch.optim.SGD(model.parameters(), lr=0.1)
    for i in range(3):
        opt.zero_grad()
        for rank in range(2):
            x = batch("cpu", seed=2 * i + rank, labelled=1.0)
            x[2].fill_(1)
            x[3][1, 11:] = 7
            with torch.no_grad():
                said = crit.answers(teacher(*x[:3])[0], x[3])
            (crit(*model(*x[:3]), x[3], x[4], said) / 2).backward()
        opt.step()
    for n, p in model.named_parameters():
        assert (a[n] == b[n]).all(), n
        # three steps of lr 0.1 on gradients under 1 whose float32 sums are
        # taken in another order: 2^-24 times the 68 tokens' terms, each step
        assert abs(a[n] - p.detach().numpy()).max() < 3 * 0.1 * 68 * 2 ** -22


@pytest.mark.timeout(600)
def test_benchmark_command_runs_with_them():
    r = subprocess.run(
        [sys.executable, os.path.join(REPO, "benchmarks", "bert_benchmark.py"),
         "--model", "bert_base", "--batch-size", "1", "--sentence-len", "12",
         "--num-warmup-batches", "1", "--num-batches-per-iter", "1",
         "--num-iters", "1", "--fused-ln", "--fused-loss",
         "--distill-top", "4"],
        capture_output=True, text=True, timeout=540, cwd=REPO)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "Total sen/sec on 1 GPU(s)" in r.stdout


# ------------------------------------------------------------------ on a GPU
@pytest.mark.gpu
@pytest.mark.parametrize("amp", [False, True])
def test_gpu_model_is_as_near_to_float64_as_the_plain_one(amp):
    """Both sides round as often, so that neither is far nearer to the
    float64 gradients than the other: a factor of 4 on the 2-norm covers the
    spread of two random sums; an error in a formula is thousands of times
    more."""
    b = batch("cuda")
    ref = small(False).double()
    said = None
    _, want = step(ref, models.BertPretrainingCriterion(VOCAB),
                   [t.cpu() for t in b])
    dist = {}
    for fused in (False, True):
        model = small(fused).cuda()
        crit = models.BertPretrainingCriterion(VOCAB, fused=fused)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=amp):
            _, g = step(model, crit, b, said)
        dist[fused] = off(g, want)
    assert dist[True] < 4 * dist[False], dist


@pytest.mark.gpu
def test_gpu_distillation_step_eager_and_captured():
    """Teacher and student with every fused operator; then the student's step
    captured and replayed on other batches, with eager work in between."""
    student, teacher = small(True).cuda(), small(True, hidden=64).cuda().eval()
    crit = models.BertDistillationCriterion(VOCAB, top=16, temperature=2.0)
    ref, ref_teacher = small(False).double(), \
        small(False, hidden=64).double().eval()
    ref_teacher.load_state_dict(teacher.state_dict())
    b = batch("cuda")
    with torch.no_grad():
        said = crit.answers(teacher(*b[:3])[0], b[3])
    loss, g = step(student, crit, b, said)
    cpu = [t.cpu() for t in b]
    with torch.no_grad():
        said64 = crit.answers(ref_teacher(*cpu[:3])[0], cpu[3])
    want, gw = step(ref, crit, cpu, said64)
    # float32 through 2 layers: sums of 96 terms, some 30 operations deep
    assert abs(loss.cpu() - want) < 30 * 96 * 2 ** -24 * want
    assert off(g, gw) < 30 * 96 * 2 ** -24

    held = [t.clone() for t in b]
    params = list(student.parameters())

    def captured():
        with torch.no_grad():
            said = crit.answers(teacher(*held[:3])[0], held[3])
        scores, seq = student(*held[:3])
        loss = crit(scores, seq, held[3], held[4], said)
        return [loss.detach(), *torch.autograd.grad(loss, params)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            captured()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = captured()
    for i in range(4):
        for t, src in zip(held, batch("cuda", seed=10 + i)):
            t.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        eager = captured()
        torch.cuda.synchronize()
        # library products may choose another kernel under capture: float32
        for a, e in zip(got, eager):
            assert (a - e).norm() <= 30 * 96 * 2 ** -24 * e.norm(), i


@pytest.mark.gpu
def test_gpu_dear_training_with_the_fused_model():
    import dear_pytorch_amd as dear
    dear.init()
    model = small(True).cuda()
    crit = models.BertPretrainingCriterion(VOCAB, fused=True)
    opt = dear.DistributedOptimizer(
        torch.optim.AdamW(model.parameters(), lr=1e-3), model=model)
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    for i in range(3):
        b = batch("cuda", seed=i)
        opt.zero_grad()
        loss = crit(*model(*b[:3]), b[3], b[4])
        loss.backward()
        opt.step()
    opt.synchronize()
    assert torch.isfinite(loss)
    for n, p in model.named_parameters():
        assert torch.isfinite(p).all() and not torch.equal(p, before[n]), n
