"""Token log probabilities and top-logit distillation against their formulas
in float64: the CPU composition, the HIP kernels (gpu-marked), what is refused.

Bounds: u is half a step of float32 (2^-24). With d_j = (z_j - m) / T:
    exp(d_j): relatively by u (3 |d_j| + 2): the difference, the product with
        log2(e) / T and that factor round once each, exp2 is good to a step;
    s, the sum: by u (3 D + 2 + chain), D = sum p |d|, where `chain` is the
        most elements that one thread adds up in float32 (V / 256 + 64);
    log s: absolutely by that, times the share of s that is not exactly 1 (the
        largest element's exp is exact and counted apart);
    sum(exp(d) d) / s: by u sum p |d| (3 |d| + 4 + chain), plus s's error.
What follows is computed in float64 and rounded to float32 once. A 16-bit
gradient adds half a step of its type, and float16 half of its smallest step
(2^-25)."""
import math

import pytest
import torch

from dear_pytorch_amd.ops.token_loss import (MAX_TOP, token_logprobs,
                                             topk_distill_loss)

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8,
        torch.float16: 2.0 ** -11}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF, NAN = math.inf, math.nan


def rounded(err, value, dtype):
    # the hardware's exp2 gives 0 for what is under 2^-126, and no factor of a
    # probability in these tests is over 2^10
    tiny = 2.0 ** -25 if dtype == F16 else 2.0 ** -116
    return err + HALF[dtype] * (value.abs() + err) + tiny


def check(got, value, err, what):
    assert got.shape == value.shape, (what, got.shape, value.shape)
    err = torch.where(torch.isfinite(err), err, 0.0)   # of rows not looked at
    value = torch.where(torch.isinf(value.to(got.dtype)),   # past its range
                        value.to(got.dtype).double(), value)
    bound = rounded(err, torch.where(torch.isfinite(value), value, 0.0),
                    got.dtype)
    got = got.double()
    fine = torch.isfinite(value)
    assert torch.equal(torch.isnan(got), torch.isnan(value)), what
    assert torch.equal(got[~fine & ~torch.isnan(value)],
                       value[~fine & ~torch.isnan(value)]), what
    off = ((got - value).abs() / bound)[fine]
    worst = off.max().item() if off.numel() else 0.0
    where = torch.where(fine, (got - value).abs() / bound, 0.0).argmax() \
        if worst > 1.0 else None
    assert worst <= 1.0, (what, worst, where, got.flatten()[where],
                          value.flatten()[where])


class Row:
    """The softmax of rows [R, V] in float64, and the bounds above."""

    def __init__(self, z, T):
        z = z.double()
        m = z.amax(-1, keepdim=True)
        self.d = (z - m) / T
        self.e = self.d.exp()
        # the largest are counted apart: 1 + 1e-20 has no digits for the rest
        best = self.d == 0
        others = torch.where(best, 0.0, self.e).sum(-1, keepdim=True) \
            + (best.sum(-1, keepdim=True) - 1)
        self.s = 1.0 + others
        self.log_s = others.log1p()
        self.lp = self.d - self.log_s
        self.p = self.e / self.s
        a = torch.where(self.e > 0, self.d.abs(), 0.0)    # no 0 * inf
        self.a = a
        self.chain = z.size(-1) / 256 + 64
        D = (self.p * a).sum(-1, keepdim=True)
        self.D = D
        loose = others / self.s                      # what is not exactly 1
        self.s_err = U * (3 * D + 2 + self.chain) * loose
        self.e2_err = U * (self.p * a * (3 * a + 4 + self.chain)) \
            .sum(-1, keepdim=True) + D * self.s_err
        h = self.log_s + D
        self.bad = torch.isnan(self.lp).any(-1, keepdim=True) \
            & ~(z == -INF) | ~torch.isfinite(m)
        self.h = torch.where(self.bad, NAN, h)
        # relative, of one probability
        self.p_rel = U * (3 * a + 4) + self.s_err


def logprobs_exact(z, tokens, top, T, ignore, ups):
    """Outputs and the logits' gradient with their bounds, rows [R, V]."""
    r = Row(z, T)
    R, V = z.shape
    keep = torch.ones(R, dtype=torch.bool, device=z.device) \
        if tokens is None else tokens != ignore
    out = {}
    lp = torch.where(r.bad, NAN, r.lp)
    coef = torch.zeros_like(lp)
    named = torch.zeros_like(lp)
    if tokens is not None:
        known = (tokens >= 0) & (tokens < V)
        at = tokens.clamp(0, V - 1)[:, None]
        v = torch.where(known, lp.gather(1, at)[:, 0], NAN)
        out["logprob"] = (torch.where(keep, v, 0.0), r.s_err[:, 0])
        up = ups.get("logprob")
        if up is not None:
            c = torch.where(known, up.double(), NAN)
            coef += c[:, None]
            named.scatter_add_(1, at, c[:, None])
    out["entropy"] = (torch.where(keep, r.h[:, 0], 0.0),
                      (r.s_err + r.e2_err)[:, 0])
    if top:
        # torch's sort on a GPU puts a NaN with a sign bit last
        ids = torch.where(torch.isnan(z), NAN, z.float()) \
            .sort(dim=-1, descending=True, stable=True)[1][:, :top]
        out["top_logprobs"] = (
            torch.where(keep[:, None], lp.gather(1, ids), -INF), r.s_err)
        out["top_ids"] = torch.where(keep[:, None], ids, -1)
        up = ups.get("top_logprobs")
        if up is not None:
            coef += up.double().sum(-1, keepdim=True)
            named.scatter_add_(1, ids, up.double())
    dh = ups["entropy"].double()[:, None] if "entropy" in ups else 0.0
    lean = torch.where(r.p > 0, r.lp + r.h, 0.0)
    spread = r.p * (coef + dh * lean)
    grad = torch.where(r.bad, NAN, (named - spread) / T)
    # the coefficients round once each and their sum up to top + 1 times; p
    # cancels against c where it is near one, so errors go by the parts
    mass = coef.abs() + named.abs().sum(-1, keepdim=True)
    abs_h = dh.abs() if torch.is_tensor(dh) else 0.0
    err = r.p * ((mass + abs_h * (r.a + r.h.abs() + r.log_s))
                 * (r.p_rel + (top + 8) * U)
                 + abs_h * (r.s_err + r.e2_err)) \
        + (top + 3) * U * named.abs()
    if ups.get("top_logprobs") is not None:
        # a sum of coefficients may cancel: its error goes by their sizes
        err = err + r.p * (top + 8) * U * ups["top_logprobs"].double().abs() \
            .sum(-1, keepdim=True)
        at_top = torch.zeros_like(lp).scatter_add_(
            1, ids, ups["top_logprobs"].double().abs())
        if "logprob" in ups:
            at_top.scatter_add_(1, at, ups["logprob"].double().abs()[:, None])
        err = err + (top + 3) * U * at_top
    out["dlogits"] = (torch.where(keep[:, None], grad, 0.0),
                      torch.where(torch.isfinite(err), err, 0.0) / T
                      * (1 + 4 * U) + 3 * U * grad.nan_to_num().abs())
    return out


def distill_exact(z, ids, teacher, T, tail, up):
    r = Row(z, T)
    R, V = z.shape
    present = ids >= 0
    live = present.any(-1, keepdim=True)
    t = teacher.double().masked_fill(~present, -INF)
    if tail:
        q = t.exp()
        rest = (1 - q.sum(-1, keepdim=True)).clamp(min=0)
    else:
        q = (t - t.amax(-1, keepdim=True)).exp().nan_to_num(0.0) \
            if not torch.isnan(teacher).any() else torch.softmax(t, -1)
        total = q.sum(-1, keepdim=True)
        q = torch.where(total > 0, q / total, q)
        rest = torch.zeros(R, 1, dtype=torch.double, device=z.device)
    at = ids.clamp(0, V - 1)
    wrong = (ids >= V).any(-1, keepdim=True)
    l_at = r.lp.gather(1, at)
    loss = torch.where(q == 0, 0.0, q * (q.log() - l_at)).sum(-1, True)
    named = torch.zeros(R, V + 1, dtype=torch.bool, device=z.device) \
        .scatter_(1, torch.where(present & (ids < V), ids, V), True)[:, :V]
    out = torch.where(named, 0.0, r.p).sum(-1, keepdim=True)
    has = (rest != 0) & (out > 0)
    loss = loss + torch.where(has, rest * (rest.log() - out.log()), 0.0)
    loss = torch.where(r.bad | wrong, NAN, loss * T * T)
    # q and rest are float64 on both sides, from the same float32 numbers
    out_err = U * (torch.where(named, 0.0, r.p) * (3 * r.a + 4 + r.chain)) \
        .sum(-1, keepdim=True) / out.clamp(min=1e-300)
    loss_err = ((q.sum(-1, True) + rest) * r.s_err
                + rest * torch.where(has, out_err, 0.0)) * T * T
    W = q.sum(-1, keepdim=True) + torch.where(has, rest, 0.0)
    shift = torch.where(has, rest / out.clamp(min=1e-300), 0.0)
    taught = torch.zeros(R, V + 1, dtype=torch.double, device=z.device) \
        .scatter_add_(1, torch.where(present & (ids < V), ids, V), q)[:, :V]
    # outside: p W - p shift, where the two may cancel
    f = torch.where(named, W, W - shift)
    g = up.double()[:, None] * T
    grad = torch.where(torch.isnan(loss), NAN, g * (r.p * f - taught))
    f_err = U * (W + 2 * f.abs()) + torch.where(
        named, 0.0, shift * (out_err + r.s_err + 2 * U))
    K = ids.size(-1)
    err = g.abs() * (r.p * (f.abs() * (r.p_rel + 4 * U) + f_err)
                     + taught * (K + 4) * U) + 3 * U * grad.nan_to_num().abs()
    return {"loss": (torch.where(live, loss, 0.0)[:, 0],
                     loss_err.nan_to_num()[:, 0]),
            "dlogits": (torch.where(live, grad, 0.0), err.nan_to_num())}


# --------------------------------------------------------------- one call each
def run_logprobs(z, tokens, ups, **kw):
    leaf = z.detach().requires_grad_(True)
    t = token_logprobs(leaf, tokens, **kw)
    got = {k: v for k, v in t._asdict().items() if v is not None}
    if ups:
        got["dlogits"], = torch.autograd.grad(
            [got[k] for k in ups], leaf, [ups[k] for k in ups])
    return {k: v.detach() for k, v in got.items()}


def compare_logprobs(z, tokens, ups, top=0, T=1.0, ignore=-1):
    got = run_logprobs(z, tokens, ups, top=top, temperature=T,
                       ignore_index=ignore)
    V = z.size(-1)
    want = logprobs_exact(
        z.reshape(-1, V), None if tokens is None else tokens.reshape(-1),
        top, T, ignore, {k: u.reshape(-1, top) if k == "top_logprobs"
                         else u.reshape(-1) for k, u in ups.items()})
    if not ups:
        want.pop("dlogits")
    assert set(got) == set(want)
    for k, v in want.items():
        if k == "top_ids":
            assert got[k].dtype == torch.int64
            assert torch.equal(got[k].reshape(-1, top), v), k
        else:
            flat = got[k].reshape(v[0].shape)
            check(flat, *v, what=k)
    with torch.no_grad():
        plain = token_logprobs(z, tokens, top=top, temperature=T,
                               ignore_index=ignore)
    for k, v in plain._asdict().items():
        assert v is None or torch.equal(v.nan_to_num(1e9),
                                        got[k].nan_to_num(1e9)), k
    return got


def run_distill(z, ids, lp, up, **kw):
    leaf = z.detach().requires_grad_(True)
    loss = topk_distill_loss(leaf, ids, lp, **kw)
    g, = torch.autograd.grad(loss, leaf, up)
    return loss.detach(), g


def compare_distill(z, ids, lp, up, T=1.0, tail=False):
    loss, g = run_distill(z, ids, lp, up, temperature=T, tail=tail)
    V, K = z.size(-1), ids.size(-1)
    want = distill_exact(z.reshape(-1, V), ids.reshape(-1, K),
                         lp.reshape(-1, K), T, tail, up.reshape(-1))
    check(loss.reshape(-1), *want["loss"], what="loss")
    check(g.reshape(-1, V), *want["dlogits"], what="dlogits")
    with torch.no_grad():
        assert torch.equal(
            topk_distill_loss(z, ids, lp, temperature=T, tail=tail)
            .nan_to_num(1e9), loss.nan_to_num(1e9))
    return loss, g


def make_logits(R, V, dtype, dev, seed=0):
    gen = torch.Generator().manual_seed(seed)
    z = torch.randn(R, V, generator=gen) * 2
    if R:
        z[torch.arange(R), torch.randint(0, V, (R,), generator=gen)] += 6
    return z.to(dtype).to(dev), gen


def make_ups(R, top, gen, dev, names=("logprob", "entropy", "top_logprobs")):
    ups = {"logprob": torch.randn(R, generator=gen),
           "entropy": torch.randn(R, generator=gen) * 0.3}
    if top:
        ups["top_logprobs"] = torch.randn(R, top, generator=gen) * 0.5
    return {k: v.to(dev) for k, v in ups.items() if k in names}


def make_teacher(z, K, T, gen, ragged=False):
    t = z.float().cpu() * 0.7
    t = (t + torch.randn(t.shape, generator=gen)) / T
    lp, ids = torch.log_softmax(t, -1).topk(K, dim=-1)
    if ragged:
        n = torch.randint(0, K + 1, (t.size(0), 1), generator=gen)
        short = torch.arange(K) >= n
        ids, lp = ids.masked_fill(short, -1), lp.masked_fill(short, -INF)
    return ids.to(z.device), lp.to(z.device)


def standard_logprobs(R, V, top, T, dtype, dev):
    z, gen = make_logits(R, V, dtype, dev, seed=R * V + top)
    tokens = torch.randint(0, V, (R,), generator=gen)
    tokens[1::3] = -1
    if R > 4:
        tokens[4] = z[4].float().argmax().item()
    compare_logprobs(z, tokens.to(dev), make_ups(R, top, gen, dev), top, T)


def standard_distill(R, V, K, T, tail, dtype, dev):
    z, gen = make_logits(R, V, dtype, dev, seed=R * V + K)
    ids, lp = make_teacher(z, K, T, gen, ragged=True)
    up = torch.rand(R, generator=gen).to(dev)
    compare_distill(z, ids, lp, up, T, tail)


def special_rows(V, dev, dtype=F32):
    """Rows where softmax, or the order of its elements, can go wrong."""
    gen = torch.Generator().manual_seed(9)
    z = torch.randn(12, V, generator=gen)
    z[0] = 0.5                                  # all equal
    z[1] = torch.arange(V) * 1e-3               # the best one last
    z[2] = -torch.arange(V) * 1e-3              # the best one first
    z[3, 1:] = -INF                             # one token is left
    z[4] = -INF                                 # none is left
    z[5, V // 2] = NAN
    z[6, V // 3] = INF
    z[7, ::2] = -INF                            # half of them are left
    z[8] = torch.where(torch.rand(V, generator=gen) < 0.5, 0.0, -0.0)
    z[9] = torch.finfo(dtype).min               # a mask by the lowest value
    z[9, V // 2] = 1.0
    z[10, 0] = 60.0                             # sure of its token
    z[11] = torch.randint(0, 3, (V,), generator=gen).float()   # many ties
    return z.to(dtype).to(dev), gen


# ------------------------------------------------------------------- on CPU
@pytest.mark.parametrize("R,V,top,T", [(5, 1, 1, 1.0), (7, 33, 5, 0.7),
                                       (3, 300, 128, 2.0), (0, 9, 2, 1.0)])
def test_cpu_logprobs(R, V, top, T):
    for dtype in (F32, BF16):
        standard_logprobs(R, V, top, T, dtype, "cpu")


@pytest.mark.parametrize("R,V,K,T", [(6, 1, 1, 1.0), (7, 33, 5, 0.7),
                                     (3, 300, 128, 2.0), (0, 9, 2, 1.0)])
@pytest.mark.parametrize("tail", [False, True])
def test_cpu_distill(R, V, K, T, tail):
    for dtype in (F32, F16):
        standard_distill(R, V, K, T, tail, dtype, "cpu")


def special_logprobs(V, top, dtype, dev):
    z, gen = special_rows(V, dev, dtype)
    tokens = torch.randint(0, V, (12,), generator=gen)
    tokens[3], tokens[10] = 0, 0
    compare_logprobs(z, tokens.to(dev), make_ups(12, top, gen, dev), top, 1.3)
    # where it is ignored a row is not looked at, whatever it holds
    got = compare_logprobs(z, torch.full((12,), -1, device=dev),
                           make_ups(12, top, gen, dev), top, 1.3)
    assert got["dlogits"].eq(0).all() and got["logprob"].eq(0).all()


def special_distill(V, K, tail, dtype, dev):
    z, gen = special_rows(V, dev, dtype)
    base = torch.randn(12, V, generator=gen)
    lp, ids = torch.log_softmax(base, -1).topk(K, -1)
    ids[3, 0] = 0
    up = torch.rand(12, generator=gen)
    compare_distill(z, ids.to(dev), lp.to(dev), up.to(dev), 1.3, tail)
    # an absent list: not looked at
    loss, g = compare_distill(z, torch.full_like(ids, -1).to(dev), lp.to(dev),
                              up.to(dev), 1.3, tail)
    assert loss.eq(0).all() and g.eq(0).all()


@pytest.mark.parametrize("V,top", [(40, 7), (40, 40)])
def test_cpu_special_rows(V, top):
    special_logprobs(V, top, F32, "cpu")
    for tail in (False, True):
        special_distill(V, top, tail, F32, "cpu")


def unknown_tokens(dev):
    z, gen = make_logits(6, 50, F32, dev)
    tokens = torch.tensor([3, 50, -7, 1 << 40, -1, 49], device=dev)
    got = compare_logprobs(z, tokens, make_ups(6, 3, gen, dev), 3)
    assert torch.isnan(got["logprob"]).tolist() == \
        [False, True, True, True, False, False]
    # without a gradient of its log probability the row is an ordinary one
    compare_logprobs(z, tokens, make_ups(6, 3, gen, dev, ("entropy",)), 3)
    # a token that is ignored may lie inside of the vocabulary
    compare_logprobs(z, tokens, make_ups(6, 3, gen, dev), 3, ignore=3)
    ids, lp = make_teacher(z, 4, 1.0, gen)
    ids[2, 1], ids[3, 3] = 50, 1 << 40
    for tail in (False, True):
        loss, _ = compare_distill(z, ids, lp, torch.ones(6, device=dev), 1.0,
                                  tail)
        assert torch.isnan(loss).tolist() == [False, False, True, True, False,
                                              False]


def test_cpu_unknown_tokens():
    unknown_tokens("cpu")


def odd_teachers(dev):
    z, gen = make_logits(7, 64, F32, dev)
    ids, lp = make_teacher(z, 6, 1.0, gen)
    up = torch.rand(7, generator=gen).to(dev)
    ids[0, 3] = ids[0, 1]                       # an id named twice
    ids[1, :] = ids[1, :1]                      # one named six times
    lp[2, 4:] = -INF                            # entries of no share
    lp[3] = -INF                                # all of them
    lp[4] = torch.tensor([0.0] + [-INF] * 5)    # sure, and nothing is left
    lp[5] = lp[5] + 3.0                         # sums up to more than one
    for tail in (False, True):
        compare_distill(z, ids, lp, up, 1.0, tail)
    # all tokens named: no tail is left, whatever rounding leaves of the sum
    w = z[:, :6].contiguous()
    every = torch.arange(6, device=dev).expand(7, 6).contiguous()
    full = torch.log_softmax(w * 0.5, -1)
    compare_distill(w, every, full, up, 1.0, True)
    # a student that gives nothing to the tokens outside: the term is left out
    masked = torch.full_like(z, -INF).scatter_(1, ids, z.gather(1, ids))
    for tail in (False, True):
        compare_distill(masked, ids, lp, up, 1.0, tail)
    # a token that the teacher names and the student rules out: +inf
    hole = z.clone()
    hole[6, ids[6, 0]] = -INF
    loss, g = compare_distill(hole, ids, lp, up, 1.0, False)
    assert loss[6] == INF and torch.isfinite(g[6]).all()


def test_cpu_odd_teachers():
    odd_teachers("cpu")


def long_lists_with_repeats(dev):
    """Up to 128 entries, some of them one token's: side by side, 64 apart,
    three times, and all of them."""
    z, gen = make_logits(6, 5000, F32, dev, seed=3)
    up = torch.rand(6, generator=gen).to(dev)
    for K in (60, 100, 128):
        ids, lp = make_teacher(z, K, 1.0, gen)
        ids[0, 1] = ids[0, 0]
        ids[1, K - 1] = ids[1, K - 65 if K > 64 else 0]
        ids[2, 7] = ids[2, K // 2] = ids[2, K - 2]
        ids[3, :] = ids[3, :1]
        ids[4, K // 2:] = ids[4, :K - K // 2].flip(0)
        for tail in (False, True):
            compare_distill(z, ids, lp - 1.0, up, 1.0, tail)


def test_cpu_long_lists_with_repeats():
    long_lists_with_repeats("cpu")


def test_gradients_against_differences():
    gen = torch.Generator().manual_seed(3)
    z = torch.randn(4, 9, generator=gen, dtype=torch.double) \
        .requires_grad_(True)
    tokens = torch.tensor([2, -1, 8, 0])

    def outs(x):
        t = token_logprobs(x, tokens, top=3, temperature=1.7)
        return t.logprob, t.entropy, t.top_logprobs[[0, 2, 3]]

    assert torch.autograd.gradcheck(outs, (z,))
    ids, lp = make_teacher(z.detach().float(), 3, 1.7, gen)
    ids[1, 2] = -1
    for tail in (False, True):
        assert torch.autograd.gradcheck(
            lambda x: topk_distill_loss(x, ids, lp, temperature=1.7,
                                        tail=tail), (z,))


def test_cpu_is_cross_entropy():
    z, _ = make_logits(20, 30, F32, "cpu")
    labels = torch.randint(0, 30, (20,))
    labels[::4] = -1
    lp = token_logprobs(z, labels).logprob
    want = torch.nn.functional.cross_entropy(z.double(), labels,
                                             ignore_index=-1, reduction="sum")
    assert abs(-lp.double().sum() - want) < 20 * 8 * U * 15


def bad_logprobs(dev="cpu"):
    z = torch.zeros(3, 5, device=dev)
    t = torch.zeros(3, dtype=torch.long, device=dev)
    return [
        (TypeError, (z.long(), t, 0)),
        (ValueError, (torch.zeros((), device=dev), None, 0)),
        (ValueError, (torch.zeros(3, 0, device=dev), None, 0)),
        (ValueError, (z, t, -1)), (ValueError, (z, t, 6)),
        (ValueError, (torch.zeros(3, 500, device=dev), t, MAX_TOP + 1)),
        (ValueError, (z, t.int(), 0)), (ValueError, (z, t[:2], 0)),
        (ValueError, (z, t[:, None], 0)),
    ]


@pytest.mark.parametrize("i", range(len(bad_logprobs())))
def test_refusals_logprobs(i):
    err, (z, t, top) = bad_logprobs()[i]
    with pytest.raises(err):
        token_logprobs(z, t, top=top)
    kernels = pytest.importorskip("dear_pytorch_amd._kernels")
    with pytest.raises(err):
        kernels.token_logprobs(z, t, top, 1.0, -1)


def bad_distill(dev="cpu"):
    z = torch.zeros(3, 5, device=dev)
    ids = torch.zeros(3, 2, dtype=torch.long, device=dev)
    lp = torch.zeros(3, 2, device=dev)
    return [
        (TypeError, (z.long(), ids, lp)), (TypeError, (z, ids, ids)),
        (ValueError, (torch.zeros(3, 0, device=dev), ids, lp)),
        (ValueError, (z, ids.int(), lp)), (ValueError, (z, ids, lp[:, :1])),
        (ValueError, (z, ids[:2], lp[:2])), (ValueError, (z, ids[0], lp[0])),
        (ValueError, (z, ids[:, :0], lp[:, :0])),
        (ValueError, (z, ids[:, :1].expand(3, MAX_TOP + 1),
                      lp[:, :1].expand(3, MAX_TOP + 1))),
    ]


@pytest.mark.parametrize("i", range(len(bad_distill())))
def test_refusals_distill(i):
    err, args = bad_distill()[i]
    with pytest.raises(err):
        topk_distill_loss(*args)
    kernels = pytest.importorskip("dear_pytorch_amd._kernels")
    with pytest.raises(err):
        kernels.topk_distill_loss(*args, 1.0, False)


def test_refusals_of_temperature_and_teacher():
    z = torch.zeros(3, 5)
    ids, lp = torch.zeros(3, 2, dtype=torch.long), torch.zeros(3, 2)
    for t in (0.0, -1.0, NAN, INF, 1e5):
        with pytest.raises(ValueError):
            token_logprobs(z, None, temperature=t)
        with pytest.raises(ValueError):
            topk_distill_loss(z, ids, lp, temperature=t)
    with pytest.raises(ValueError, match="detach"):
        topk_distill_loss(z, ids, lp.requires_grad_(True))


def test_most_entries():
    kernels = pytest.importorskip("dear_pytorch_amd._kernels")
    assert kernels.max_top == MAX_TOP


# ------------------------------------------------------------------ on a GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("R,V,top,T", [
    (1, 1, 1, 1.0), (5, 2, 2, 1.0), (9, 5, 0, 0.7), (4, 63, 63, 1.0),
    (33, 257, 8, 2.0), (6, 1000, 128, 1.0), (5, 4097, 64, 4.0),
    (1, 30528, 8, 1.0), (40, 30522, 5, 1.0), (3, 30528, 128, 1.5),
    (2, 70001, 33, 1.0), (3, 131075, 128, 1.0), (300, 129, 1, 1.0),
    (2, 600011, 20, 1.0),
    # rows of several pieces and no alternatives; more lists than are held at
    # once; enough rows for the longest pieces
    (2, 70001, 0, 1.0), (300, 30528, 0, 1.0), (2, 600011, 128, 1.0),
    (300, 40009, 17, 1.0), (150, 70001, 64, 1.0)])
def test_gpu_logprobs(R, V, top, T, dtype):
    standard_logprobs(R, V, top, T, dtype, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("R,V,top,T", [
    # a block to each row, finished there and, of more rows, apart
    (2, 30528, 0, 1.0), (255, 9001, 128, 1.0), (4200, 300, 5, 1.0),
    (4200, 300, 0, 1.0), (1100, 1500, 40, 1.0), (1100, 5001, 0, 2.0),
    (600, 16001, 20, 1.0),
    # more slices than a wave has lanes
    (1, 2200001, 128, 1.0), (1, 2200001, 7, 1.0), (1, 2200001, 0, 1.0)])
def test_gpu_logprobs_blocks(R, V, top, T, dtype):
    standard_logprobs(R, V, top, T, dtype, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("V", [262144, 280001])
def test_gpu_equal_lists(V):
    """Slices that are alike but for one that is worse: next to nothing of
    their lists can be left out."""
    gen = torch.Generator().manual_seed(5)
    one = torch.randn(2, 16384, generator=gen)
    z = one.repeat(1, 18)[:, :V].contiguous()
    z[:, 16384:32768] -= 30.0
    tokens = torch.tensor([7, V - 1]).cuda()
    compare_logprobs(z.cuda(), tokens, make_ups(2, 128, gen, "cuda"), 128, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("R,V,K,T", [
    (2, 1, 1, 1.0), (5, 2, 2, 1.0), (9, 5, 3, 0.7), (4, 63, 63, 1.0),
    (33, 257, 8, 2.0), (6, 1000, 128, 1.0), (1, 30528, 8, 1.0),
    (40, 30522, 5, 1.0), (3, 30528, 128, 4.0), (3, 131075, 64, 1.0),
    (2, 600011, 20, 1.0)])
def test_gpu_distill(R, V, K, T, tail, dtype):
    standard_distill(R, V, K, T, tail, dtype, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V,top", [(40, 40), (300, 9), (5000, 128),
                                   (30522, 20), (140000, 5)])
def test_gpu_special_rows(V, top, dtype):
    special_logprobs(V, top, dtype, "cuda")
    for tail in (False, True):
        special_distill(V, top, tail, dtype, "cuda")


@pytest.mark.gpu
def test_gpu_unknown_tokens():
    unknown_tokens("cuda")


@pytest.mark.gpu
def test_gpu_odd_teachers():
    odd_teachers("cuda")


@pytest.mark.gpu
def test_gpu_long_lists_with_repeats():
    long_lists_with_repeats("cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("names", [("logprob",), ("entropy",),
                                   ("top_logprobs",),
                                   ("logprob", "top_logprobs")])
def test_gpu_some_gradients(names):
    z, gen = make_logits(9, 700, F32, "cuda")
    tokens = torch.randint(0, 700, (9,), generator=gen)
    tokens[2] = z[2].argmax().item()         # a token that is in its own top
    compare_logprobs(z, tokens.cuda(), make_ups(9, 6, gen, "cuda", names), 6)
    if "logprob" not in names:
        compare_logprobs(z, None, make_ups(9, 6, gen, "cuda", names), 6)


@pytest.mark.gpu
def test_gpu_shapes_and_strides():
    z, gen = make_logits(12, 210, F32, "cuda")
    tokens = torch.randint(0, 150, (12,), generator=gen).cuda()
    ups = make_ups(12, 4, gen, "cuda")
    for v in (z[:, 3:190], z.half()[:, 1:180], z[:, ::1][:, :151],
              z.t().contiguous().t(), z[:, ::2][:, :105].repeat(1, 2),
              z[:1].expand(12, 210), z[:, ::1].as_strided((12, 160), (3, 1))):
        compare_logprobs(v, tokens, ups, 4)
        ids, lp = make_teacher(v.contiguous(), 5, 1.0, gen)
        compare_distill(v, ids, lp, ups["entropy"].abs(), 1.0, True)
    # columns that are two apart, odd leading shapes, one row
    compare_logprobs(z[:, ::2], tokens % 100, ups, 4)
    cut = lambda t: t.reshape(3, 4, *t.shape[1:])
    compare_logprobs(cut(z), cut(tokens),
                     {k: cut(u) for k, u in ups.items()}, 4)
    compare_logprobs(cut(z).transpose(0, 1), cut(tokens).t(),
                     {k: cut(u).transpose(0, 1) for k, u in ups.items()}, 4)
    ids, lp = make_teacher(z, 5, 1.0, gen)
    compare_distill(cut(z).transpose(0, 1), cut(ids).transpose(0, 1),
                    cut(lp).transpose(0, 1),
                    torch.ones((), device="cuda").expand(4, 3), 1.0, False)
    one = token_logprobs(z[5], tokens[5], top=2)
    assert one.logprob.shape == () and one.top_ids.shape == (2,)
    assert torch.equal(one.top_ids, token_logprobs(z, tokens, top=2)
                       .top_ids[5])
    half = lp.bfloat16()
    assert torch.equal(topk_distill_loss(z, ids, half),
                       topk_distill_loss(z, ids, half.float()))


@pytest.mark.gpu
def test_gpu_no_rows():
    z = torch.zeros(0, 40, device="cuda")
    tokens = torch.zeros(0, dtype=torch.long, device="cuda")
    got = run_logprobs(z, tokens, {"logprob": z[:, 0]}, top=3)
    assert got["top_ids"].shape == (0, 3) and got["dlogits"].shape == (0, 40)
    loss, g = run_distill(z, tokens[:, None], z[:, :1], z[:, 0])
    assert loss.shape == (0,) and g.shape == (0, 40)


@pytest.mark.gpu
def test_gpu_bad_rows_stay_alone():
    z, gen = make_logits(12, 3000, F32, "cuda")
    bad = z.clone()
    bad[2, 5], bad[6, 0], bad[9] = NAN, INF, -INF
    tokens = torch.randint(0, 3000, (12,), generator=gen).cuda()
    ups = make_ups(12, 3, gen, "cuda")
    a, b = (run_logprobs(x, tokens, ups, top=3) for x in (z, bad))
    keep = [i for i in range(12) if i not in (2, 6, 9)]
    for k in a:
        assert torch.equal(a[k][keep], b[k][keep]), k
    assert torch.isnan(b["dlogits"][[2, 6, 9]]).all()


@pytest.mark.gpu
def test_gpu_same_call_same_bits():
    z, gen = special_rows(30522, "cuda", BF16)
    tokens = torch.randint(0, 30522, (12,), generator=gen).cuda()
    ups = make_ups(12, 128, gen, "cuda")
    ids, lp = make_teacher(make_logits(12, 30522, BF16, "cuda")[0], 128, 1.0,
                           gen)
    up = torch.rand(12, generator=gen).cuda()
    first = None
    for _ in range(4):
        got = run_logprobs(z, tokens, ups, top=128)
        got["loss"], got["dz"] = run_distill(z, ids, lp, up, tail=True)
        got = {k: v.nan_to_num(1e9) for k, v in got.items()}
        first = first or got
        assert all(torch.equal(first[k], got[k]) for k in got)


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    V, R = 30528, 70400                       # over 2^31 elements
    z = torch.empty(R, V, dtype=BF16, device="cuda").fill_(0.25)
    ends, gen = make_logits(8, V, BF16, "cuda")
    z[:4], z[-4:] = ends[:4], ends[4:]
    tokens = torch.full((R,), -1, device="cuda")
    rows = [0, 1, 2, 3, R - 4, R - 3, R - 2, R - 1]
    tokens[rows] = torch.randint(0, V, (8,), generator=gen).cuda()
    up = torch.zeros(R, device="cuda")
    up[rows] = torch.randn(8, generator=gen).cuda()
    got = run_logprobs(z, tokens, {"logprob": up}, top=4)
    want = logprobs_exact(ends, tokens[rows], 4, 1.0, -1,
                          {"logprob": up[rows]})
    assert torch.equal(got["top_ids"][rows], want["top_ids"])
    for k in ("logprob", "entropy", "top_logprobs", "dlogits"):
        check(got[k][rows], *want[k], what=k)
    assert got["dlogits"][4:-4].eq(0).all()
    ids = torch.full((R, 3), -1, device="cuda")
    lp = torch.full((R, 3), -INF, device="cuda")
    ids[rows], lp[rows] = make_teacher(ends, 3, 1.0, gen)
    del got
    loss, g = run_distill(z, ids, lp, up, tail=True)
    want = distill_exact(ends, ids[rows], lp[rows], 1.0, True, up[rows])
    check(loss[rows], *want["loss"], what="loss")
    check(g[rows], *want["dlogits"], what="dlogits")


@pytest.mark.gpu
def test_gpu_streams_and_graph():
    z, gen = make_logits(17, 5001, F32, "cuda")
    tokens = torch.randint(0, 5001, (17,), generator=gen)
    tokens[3] = -1
    tokens = tokens.cuda()
    ups = make_ups(17, 9, gen, "cuda")
    ids, lp = make_teacher(z, 9, 1.0, gen)
    up = torch.rand(17, generator=gen).cuda()

    def both(z, tokens, ids, lp):
        got = run_logprobs(z, tokens, ups, top=9)
        got["loss"], got["dz"] = run_distill(z, ids, lp, up, tail=True)
        return got

    want = both(z, tokens, ids, lp)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(z, tokens, ids, lp)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(want[k], got[k]) for k in want)
    held = [t.clone() for t in (z, tokens, ids, lp)]
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both(*held)
        graphs.append((graph, out))
    for i in range(4):
        for t, src in zip(held, (z, tokens, ids, lp)):
            t.copy_(torch.roll(src, i, 0))
        eager = both(*held)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(out[k], eager[k]) for k in eager), i


@pytest.mark.gpu
def test_gpu_capture_beside_a_live_eager_graph_is_refused():
    z, gen = make_logits(5, 300, F32, "cuda")
    z.requires_grad_(True)
    ids, lp = make_teacher(z.detach(), 4, 1.0, gen)
    for loss in (lambda: token_logprobs(z, ids[:, 0].contiguous()).logprob,
                 lambda: topk_distill_loss(z, ids, lp)):
        alive, up = loss(), torch.ones(5, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = loss()
            with pytest.raises(RuntimeError, match="alive"):
                torch.autograd.grad(y, z, up)
        want, = torch.autograd.grad(alive, z, up)
        del alive, y
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, = torch.autograd.grad(loss(), z, up)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


@pytest.mark.gpu
def test_gpu_second_derivative_is_refused():
    z = torch.randn(3, 9, device="cuda", requires_grad=True)
    tokens = torch.zeros(3, dtype=torch.long, device="cuda")
    for out in (token_logprobs(z, tokens).logprob,
                topk_distill_loss(z, tokens[:, None],
                                  torch.zeros(3, 1, device="cuda"))):
        g, = torch.autograd.grad(out.square().sum(), z, create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            g.sum().backward()


@pytest.mark.gpu
def test_gpu_refuses_what_the_kernel_lacks():
    z = torch.zeros(2, 8, device="cuda")
    t = torch.zeros(2, dtype=torch.long)
    with pytest.raises(TypeError):
        token_logprobs(z.double(), None)
    with pytest.raises(ValueError):
        token_logprobs(z, t)
    with pytest.raises(TypeError):
        topk_distill_loss(z, t.cuda()[:, None], z[:, :1].double())
    with pytest.raises(ValueError):
        topk_distill_loss(z, t[:, None], torch.zeros(2, 1))


@pytest.mark.gpu
def test_gpu_teacher_to_student():
    """What a teacher writes down goes into the student's loss as it is."""
    teacher, gen = make_logits(24, 30528, BF16, "cuda", seed=1)
    student, _ = make_logits(24, 30528, F32, "cuda", seed=2)
    labels = torch.randint(0, 30528, (24,), generator=gen)
    labels[::5] = -1
    labels = labels.cuda()
    said = token_logprobs(teacher, labels, top=32, temperature=2.0)
    for tail in (False, True):
        loss, g = compare_distill(student, said.top_ids, said.top_logprobs,
                                  torch.ones(24, device="cuda"), 2.0, tail)
        assert loss[::5].eq(0).all() and g[::5].eq(0).all()
    # a student that is the teacher has nothing to learn: the loss is off by
    # the rounding of 32 log probabilities to float32 (u of up to 20 each)
    same = topk_distill_loss(teacher, said.top_ids, said.top_logprobs,
                             temperature=2.0, tail=True)
    assert same.abs().max() < 4 * 4 * 40 * U
