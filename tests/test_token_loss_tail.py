"""Distillation with a tail whose tokens lie far below the teacher's entries,
against the definition in log space in float64.

With m_o the largest logit outside of the entries, d_o = (z - m_o) / T and
S = sum exp(d_o) over the outside:
    log p_t = (m_o - m) / T + log S - log s
    dz_j    = T dloss (W p_j - q_t exp(d_o) / S)       outside
    dz_j    = T dloss (W p_j - sum q_k)                named
Bounds (u is half a step of float32, 2^-24): exp(d_o) is off relatively by
u (3 |d_o| + 2), S by o = u sum exp(d_o) (3 |d_o| + 4 + chain) / S with `chain`
the elements that one thread adds up (V / 256 + 64). The entries' own sums are
float64 on both sides, so s is off relatively by o p_t where there is a tail
and by its own u (3 D + 4 + chain) without one. The rest is float64, 2^-48 of
its parts at the worst, and rounds to float32 once; dloss T, its products with
the row's factor and with exp(d_o) round once each. exp2 gives 0 under 2^-126.
"""
import math

import pytest
import torch

from dear_pytorch_amd.ops.token_loss import topk_distill_loss
from test_token_loss import BF16, F16, F32, INF, U, rounded, run_distill

DTYPES = [F32, BF16, F16]
GAPS = [3.0, 60.0, 80.0, 87.5, 90.0, 100.0, 110.0, 200.0, 700.0, 3000.0]
SLACK = 2.0 ** -48


def exact(z, ids, teacher, T, tail, up):
    """Loss and gradient with their bounds; rows with a distribution, ids
    inside of the vocabulary, each row with an entry."""
    z = z.double()
    R, V = z.shape
    chain = V / 256 + 64
    present = ids >= 0
    t = teacher.double().masked_fill(~present, -INF)
    q = t.exp() if tail else torch.softmax(t, -1)
    sure = q.sum(-1, keepdim=True)
    rest = (1 - sure).clamp(min=0) if tail else torch.zeros_like(sure)
    m = z.amax(-1, keepdim=True)
    d = (z - m) / T
    best = d == 0          # log s, with the digits of a sure row
    log_s = (torch.where(best, 0.0, d.exp()).sum(-1, keepdim=True)
             + (best.sum(-1, keepdim=True) - 1)).log1p()
    lp = d - log_s
    p = lp.exp()
    named = torch.zeros(R, V + 1, dtype=torch.bool, device=z.device) \
        .scatter_(1, torch.where(present, ids, V), True)[:, :V]
    apart = named if tail else torch.zeros_like(named)
    zo = z.masked_fill(apart, -INF)
    mo = zo.amax(-1, keepdim=True)
    some = mo > -INF
    do = torch.where(apart, -INF, (z - mo.masked_fill(~some, 0.0)) / T)
    eo = do.exp()
    S = torch.where(some, eo.sum(-1, keepdim=True), 1.0)
    ao = torch.where(eo > 0, do.abs(), 0.0)
    o_err = U * (eo * (3 * ao + 4 + chain)).sum(-1, keepdim=True) / S
    pt = p.masked_fill(apart, 0.0).sum(-1, keepdim=True)
    s_err = o_err * pt
    l_at = lp.gather(1, ids.clamp(min=0))
    parts = torch.where(q > 0, q * (t - l_at) if tail else
                        q * (torch.log_softmax(t, -1) - l_at), 0.0)
    loss, size = parts.sum(-1, True), parts.abs().sum(-1, True)
    has = some & (rest > 0)
    log_pt = torch.where(some, (mo - m) / T + S.log(), 0.0) - log_s
    gap = torch.where(has, rest * (rest.log() - log_pt), 0.0)
    loss, size = loss + gap, size + gap.abs()
    W = sure + torch.where(has, rest, 0.0)
    loss_err = T * T * (W * s_err + torch.where(has, rest, 0.0) * o_err
                        + SLACK * size)
    g = up.double()[:, None].abs() * T
    taught = torch.zeros(R, V + 1, dtype=torch.double, device=z.device) \
        .scatter_add_(1, torch.where(present, ids, V), q)[:, :V]
    B = torch.where(has & ~apart, rest * eo / S, 0.0)
    grad = up.double()[:, None] * T * (W * p - taught - B)
    out_err = (W * p - B).abs() * U * (3 * ao + 7) + W * p * s_err + B * o_err \
        + 2.0 ** -125 * (W * pt + rest) / S
    in_err = (W * p - taught).abs() * 4 * U + W * p * s_err \
        + SLACK * (W * p + taught)
    err = g * torch.where(named, in_err, out_err)
    return {"loss": ((loss * T * T)[:, 0], loss_err[:, 0]),
            "dlogits": (grad, err)}


def check(got, value, err, what):
    assert got.shape == value.shape, what
    value = torch.where(torch.isinf(value.to(got.dtype)),   # past its range
                        value.to(got.dtype).double(), value)
    fine = torch.isfinite(value)
    assert torch.isfinite(err[fine]).all(), what    # a bound that says something
    bound = rounded(err, torch.where(fine, value, 0.0), got.dtype)
    got = got.double()
    assert torch.equal(got[~fine], value[~fine]), what
    off = torch.where(fine, (got - value).abs() / bound, 0.0)
    i = off.argmax()
    assert (off <= 1.0).all(), (what, off.flatten()[i], i, got.flatten()[i],
                                value.flatten()[i])


def compare(z, ids, lp, up, T, tail):
    loss, g = run_distill(z, ids, lp, up, temperature=T, tail=tail)
    want = exact(z, ids, lp, T, tail, up)
    check(loss, *want["loss"], what="loss")
    check(g, *want["dlogits"], what="dlogits")
    with torch.no_grad():
        assert torch.equal(topk_distill_loss(z, ids, lp, temperature=T,
                                             tail=tail), loss)
    return loss, g


def ups(n, dev):
    return torch.tensor([1.0, 0.0, 65536.0, 0.25])[torch.arange(n) % 4].to(dev)


def far_rows(V, K, T, dtype, dev, where="all"):
    """A row for each gap: the entries above all others by that many T. The
    others are everywhere, or only among the first or the last tokens while
    those between are ruled out."""
    gen = torch.Generator().manual_seed(V + K)
    R = len(GAPS)
    z = torch.randn(R, V, generator=gen) * T
    if where == "first":
        z[:, max(1, V // 8):] = -INF
    elif where == "last":
        z[:, :V - max(1, V // 8)] = -INF
    ids = torch.stack([torch.randperm(V, generator=gen)[:K]
                       for _ in range(R)])
    if where != "all":     # the largest one at the other end
        ids[:, 0] = V - 1 if where == "first" else 0
        ids[:, 1:] = torch.where(ids[:, 1:] == ids[:, :1], 1, ids[:, 1:])
    above = torch.tensor(GAPS)[:, None] + torch.rand(R, K, generator=gen)
    z.scatter_(1, ids, 4 * T + above * T)
    share = torch.rand(R, K, generator=gen) + 0.1
    lp = (share / share.sum(-1, True) * 0.7).log()
    return z.to(dtype).to(dev), ids.to(dev), lp.to(dev)


def far(V, K, T, dtype, dev, where="all"):
    z, ids, lp = far_rows(V, K, T, dtype, dev, where)
    for tail in (True, False):
        loss, g = compare(z, ids, lp, ups(len(GAPS), dev), T, tail)
        assert torch.isfinite(loss).all()
        if tail:
            assert (loss > 0).all()
            assert (g[1::4] == 0).all() and not (g[0::4] == 0).all(-1).any()


def lowest(V, dtype, dev):
    """All tokens outside masked by the type's lowest value: the student still
    gives them something, in the definition. Next to that, one of them is
    left, and nothing is."""
    gen = torch.Generator().manual_seed(V)
    z = torch.full((4, V), torch.finfo(dtype).min)
    ids = torch.randint(0, V, (4, 1), generator=gen)
    z[2], z[3] = -INF, -INF
    z[2, (ids[2, 0] + 1) % V] = -90.0
    z.scatter_(1, ids, torch.tensor([[1.0], [100.0], [50.0], [1.0]]))
    lp = torch.full((4, 1), math.log(0.75))
    z, ids, lp = z.to(dtype).to(dev), ids.to(dev), lp.to(dev)
    loss, g = compare(z, ids, lp, torch.ones(4, device=dev), 1.0, True)
    # nothing outside: the term is left out, and what is named is certain
    assert abs(loss[3].item() - 0.75 * math.log(0.75)) < 1e-6
    assert (g[3] == 0).all()


def one_and_many(V, dtype, dev):
    """A row alone and one of many are cut in other ways: the same numbers,
    within the bounds."""
    z, ids, lp = far_rows(V, 3, 0.1, dtype, dev)
    for i in (2, 5, 8):
        one = [t[i:i + 1] for t in (z, ids, lp)]
        compare(*one, torch.ones(1, device=dev), 0.1, True)
        many = [t.repeat(300, 1) for t in one]
        loss, _ = compare(*many, torch.ones(300, device=dev), 0.1, True)
        assert (loss == loss[0]).all()


@pytest.mark.parametrize("where", ["all", "first", "last"])
@pytest.mark.parametrize("V,K,T", [(4, 1, 1.0), (40, 5, 0.1), (300, 17, 2.0)])
def test_cpu_far(V, K, T, where):
    for dtype in DTYPES:
        far(V, K, T, dtype, "cpu", where)


def test_cpu_lowest_and_one_of_many():
    for dtype in DTYPES:
        lowest(40, dtype, "cpu")
        one_and_many(300, dtype, "cpu")


def test_cpu_a_tail_in_its_numbers():
    """[100, 0, 0, 0] against an entry of one half for the first: by hand."""
    z = torch.tensor([[100.0, 0, 0, 0], [10.0, 0, 0, 0]])
    ids, lp = torch.zeros(2, 1, dtype=torch.long), torch.full((2, 1), 0.5).log()
    loss, g = run_distill(z[:1], ids[:1], lp[:1], torch.ones(1), tail=True)
    # 1/2 log 1/2 + 1/2 (log 1/2 - (log 3 - 100))
    assert abs(loss[0].item() - (math.log(0.5) + 50 - 0.5 * math.log(3))) < 1e-5
    assert (g[0] - torch.tensor([0.5] + [-1 / 6] * 3)).abs().max() < 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("where", ["all", "first", "last"])
@pytest.mark.parametrize("V,K,T", [
    (4, 1, 1.0), (40, 5, 0.1), (300, 17, 2.0), (5000, 128, 0.05),
    (30528, 32, 1.0), (30528, 100, 0.1), (70001, 9, 1.0), (131075, 1, 0.5)])
def test_gpu_far(V, K, T, where, dtype):
    far(V, K, T, dtype, "cuda", where)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [2, 40, 9000, 30528, 70001])
def test_gpu_lowest(V, dtype):
    lowest(V, dtype, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [300, 30528])
def test_gpu_one_of_many(V, dtype):
    one_and_many(V, dtype, "cuda")


@pytest.mark.gpu
def test_gpu_a_tail_is_the_cpu_paths():
    z, ids, lp = far_rows(30528, 12, 1.0, F32, "cpu")
    ids[3, 4:] = ids[3, :1]                     # named more than once
    ids[6, 6:] = -1
    up = ups(len(GAPS), "cpu")
    loss, g = run_distill(z, ids, lp, up, tail=True)
    got, dz = run_distill(z.cuda(), ids.cuda(), lp.cuda(), up.cuda(),
                          tail=True)
    want = exact(z, ids, lp, 1.0, True, up)
    for a, b, key in ((got, loss, "loss"), (dz, g, "dlogits")):
        check(a.cpu(), *want[key], what=key)
        check(b, *want[key], what=key)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])       # float16 ends at 65504
@pytest.mark.parametrize("where", ["all", "last"])
@pytest.mark.parametrize("V,K,T", [
    (40, 3, 1e-4), (30528, 9, 1e-4), (40, 3, 1e4), (30528, 70, 1e4)])
def test_gpu_far_at_the_ends_of_the_temperature(V, K, T, where, dtype):
    far(V, K, T, dtype, "cuda", where)
