"""Cases of the language-model operators: layer norm with a residual, log
probabilities of given tokens with entropy and top alternatives, and
distillation from a teacher's top logits — each in a plain form made of
elementary torch operations, and through the package's entry points.

A case is a dict of plain values:

    op       "norm" | "logprobs" | "distill"
    rows     tokens in the batch (batch size times sequence length)
    width    hidden size ("norm") or vocabulary ("logprobs", "distill")
    dtype    "fp32" | "bf16" | "fp16"; "norm" also has "amp": a bf16 branch
             added to an fp32 residual stream, with fp32 weights
    grad     whether the pass is a training pass (forward and backward)
    ...      and what each operator takes besides (see listed())
"""
import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16,
           "fp16": torch.float16, "amp": torch.bfloat16}
_EPS = 1e-12          # the layer norms of the BERT configurations
_DEVICE = "cuda"


def listed():
    return [
        # the hidden state of one token, the smallest call of BERT-Base: latency
        {"name": "norm-one-token", "op": "norm", "rows": 1, "width": 768,
         "dtype": "fp32", "residual": True, "grad": False},
        # one of BERT-Base's layer norms in fp32 training, 32 x 128 tokens
        {"name": "norm-base-train", "op": "norm", "rows": 4096, "width": 768,
         "dtype": "fp32", "residual": True, "grad": True},
        # BERT-Large under bf16 autocast, 32 x 512 tokens
        {"name": "norm-large-amp-train", "op": "norm", "rows": 16384,
         "width": 1024, "dtype": "amp", "residual": True, "grad": True},
        # an odd width and a ragged number of tokens, no residual
        {"name": "norm-odd-train", "op": "norm", "rows": 5077, "width": 1011,
         "dtype": "fp16", "residual": False, "grad": True},
        # the answer for one masked token with its alternatives: latency
        {"name": "logprobs-one-token", "op": "logprobs", "rows": 1,
         "width": 30528, "dtype": "fp32", "labelled": 1.0, "top": 8,
         "temperature": 1.0, "entropy_grad": False, "grad": False},
        # the masked-token loss of 32 x 128 tokens, 15 % of them labelled
        {"name": "logprobs-mlm-train", "op": "logprobs", "rows": 4096,
         "width": 30528, "dtype": "fp32", "labelled": 0.15, "top": 0,
         "temperature": 1.0, "entropy_grad": False, "grad": True},
        # a teacher that writes down its alternatives for every token
        {"name": "logprobs-teacher", "op": "logprobs", "rows": 4096,
         "width": 30528, "dtype": "bf16", "labelled": 1.0, "top": 32,
         "temperature": 2.0, "entropy_grad": False, "grad": False},
        # few rows, a long odd vocabulary, an entropy bonus and gradients of
        # the alternatives
        {"name": "logprobs-long-train", "op": "logprobs", "rows": 167,
         "width": 100003, "dtype": "fp16", "labelled": 0.9, "top": 20,
         "temperature": 1.0, "entropy_grad": True, "grad": True},
        # a small classifier head learning from another one
        {"name": "distill-small-train", "op": "distill", "rows": 8,
         "width": 1000, "dtype": "fp32", "labelled": 1.0, "top": 8,
         "temperature": 2.0, "tail": False, "ragged": False, "grad": True},
        # the labelled tokens of a 32 x 128 batch, gathered by the caller
        {"name": "distill-mlm-train", "op": "distill", "rows": 614,
         "width": 30528, "dtype": "fp32", "labelled": 1.0, "top": 64,
         "temperature": 2.0, "tail": False, "ragged": False, "grad": True},
        # every token of a 32 x 128 batch, the rest of the vocabulary as a tail
        {"name": "distill-tail-train", "op": "distill", "rows": 4096,
         "width": 30528, "dtype": "bf16", "labelled": 1.0, "top": 32,
         "temperature": 1.0, "tail": True, "ragged": False, "grad": True},
        # the unpadded vocabulary, lists of different lengths, unlabelled rows
        {"name": "distill-odd-train", "op": "distill", "rows": 331,
         "width": 30522, "dtype": "fp16", "labelled": 0.8, "top": 17,
         "temperature": 1.5, "tail": True, "ragged": True, "grad": True},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high + 1)))
    return max(low, min(high, int(v)))


def draw(rng):
    op = rng.choice(["norm", "logprobs", "distill"])
    grad = rng.random() < 0.7
    if op == "norm":
        width = _spread(rng, 16, 8192)
        rows = _spread(rng, 1, min(16384, (1 << 24) // width))
        return {"op": op, "rows": rows, "width": width,
                "dtype": rng.choice(["fp32", "bf16", "fp16", "amp"]),
                "residual": True if rng.random() < 0.6 else False,
                "grad": grad}
    width = _spread(rng, 100, 131072)
    rows = _spread(rng, 1, min(4096, (1 << 25) // width))
    case = {"op": op, "rows": rows, "width": width,
            "dtype": rng.choice(["fp32", "bf16", "fp16"]),
            "labelled": rng.choice([1.0, 1.0, 0.85, 0.15]),
            "temperature": rng.choice([1.0, 1.0, 0.7, 2.0, 4.0]),
            "grad": grad}
    if op == "logprobs":
        case["top"] = rng.choice([0, _spread(rng, 1, 64)])
        case["entropy_grad"] = rng.random() < 0.4
    else:
        case["top"] = _spread(rng, 1, min(128, width))
        case["tail"] = rng.random() < 0.5
        case["ragged"] = rng.random() < 0.4
    return case


# ---------------------------------------------------------------- the inputs
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=_DEVICE)


def _logits(gen, rows, width, dtype):
    """Logits as a trained head gives them: a spread of a few units, and a
    favourite that stands out in most rows."""
    z = _randn(gen, rows, width).mul_(2.0)
    at = torch.randint(0, width, (rows, 1), generator=gen, device=_DEVICE)
    return z.scatter_add_(1, at, _randn(gen, rows, 1).abs_().mul_(6.0)) \
        .to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=_DEVICE).manual_seed(seed)
    rows, width, dtype = case["rows"], case["width"], _DTYPES[case["dtype"]]
    s = {"case": dict(case)}
    if case["op"] == "norm":
        wide = torch.float32 if case["dtype"] == "amp" else dtype
        # hidden states: an offset a token, a few channels that are far larger
        loud = 1.0 + 6.0 * (torch.rand(width, generator=gen,
                                       device=_DEVICE) < 0.01)
        s["x"] = (_randn(gen, rows, width) * loud
                  + _randn(gen, rows, 1)).to(dtype)
        if case["residual"]:
            s["residual"] = (_randn(gen, rows, width) * loud).to(wide)
        # where there is no residual stream the branch gives its own type
        out = wide if case["residual"] else dtype
        s["weight"] = (1.0 + 0.1 * _randn(gen, width)).to(wide)
        s["bias"] = (0.1 * _randn(gen, width)).to(wide)
        if case["grad"]:
            s["dy"] = _randn(gen, rows, width).to(out)
            for k in ("x", "residual", "weight", "bias"):
                if k in s:
                    s[k].requires_grad_(True)
        return s
    s["logits"] = _logits(gen, rows, width, dtype)
    labelled = torch.rand(rows, generator=gen, device=_DEVICE) \
        < case["labelled"]
    if case["op"] == "logprobs":
        tokens = torch.randint(0, width, (rows,), generator=gen,
                               device=_DEVICE)
        # the favourite is the right one in half of the rows
        best = s["logits"].argmax(-1)
        tokens = torch.where(torch.rand(rows, generator=gen, device=_DEVICE)
                             < 0.5, best, tokens)
        s["tokens"] = torch.where(labelled, tokens, -1)
        if case["grad"]:
            s["d_logprob"] = _randn(gen, rows)
            if case["entropy_grad"]:
                s["d_entropy"] = 0.1 * _randn(gen, rows)
                if case["top"]:
                    s["d_top"] = 0.1 * _randn(gen, rows, case["top"])
    else:
        # the teacher agrees with the student in part
        k = case["top"]
        z = s["logits"].float().mul_(0.7).add_(_randn(gen, rows, width))
        z.div_(case["temperature"])
        val, ids = z.topk(k, dim=-1)
        lp = val - z.logsumexp(-1, keepdim=True)
        del z
        if case["ragged"]:
            n = torch.randint(1, k + 1, (rows, 1), generator=gen,
                              device=_DEVICE)
            short = torch.arange(k, device=_DEVICE) >= n
            ids = ids.masked_fill(short, -1)
            lp = lp.masked_fill(short, -math.inf)
        s["top_ids"] = ids.masked_fill(~labelled[:, None], -1)
        s["top_logprobs"] = lp.masked_fill(~labelled[:, None], -math.inf)
        if case["grad"]:
            s["d_loss"] = torch.rand(rows, generator=gen, device=_DEVICE)
    if case["grad"]:
        s["logits"].requires_grad_(True)
    return s


# ------------------------------------------------------------ the plain forms
def _plain_norm(s):
    x, w, b = s["x"], s["weight"].float(), s["bias"].float()
    z = x.float()
    out = x.dtype
    if "residual" in s:
        z = z + s["residual"].float()
        out = s["residual"].dtype
    mean = z.mean(-1, keepdim=True)
    d = z - mean
    rstd = (d * d).mean(-1, keepdim=True).add(_EPS).rsqrt()
    n = d * rstd
    y = {"y": (n * w + b).to(out)}
    if "dy" in s:
        dy = s["dy"].float()
        g = dy * w
        dz = rstd * (g - g.mean(-1, keepdim=True)
                     - n * (g * n).mean(-1, keepdim=True))
        y["dx"] = dz.to(x.dtype)
        if "residual" in s:
            y["dresidual"] = dz.to(s["residual"].dtype)
        y["dweight"] = (dy * n).sum(0).to(s["weight"].dtype)
        y["dbias"] = dy.sum(0).to(s["bias"].dtype)
    return y


def _plain_softmax(logits, temperature):
    """Distance to the row's largest logit, exp of it, and the sum: elements
    in 32 bits, sums in 64, so that the log probability of a token that the
    row is sure of keeps its digits."""
    z = logits.float()
    d = (z - z.amax(-1, keepdim=True)) / temperature
    e = d.exp()
    return d, e, e.sum(-1, keepdim=True, dtype=torch.double)


def _plain_logprobs(s):
    c, logits, tokens = s["case"], s["logits"], s["tokens"]
    d, e, total = _plain_softmax(logits, c["temperature"])
    log_total = total.log()
    keep = tokens >= 0
    at = tokens.clamp(min=0)[:, None]
    entropy = (log_total - (e * d).sum(-1, keepdim=True, dtype=torch.double)
               / total)[:, 0]
    logprob = (d.gather(1, at).double() - log_total)[:, 0]
    r = {"logprob": torch.where(keep, logprob, 0.0).float(),
         "entropy": torch.where(keep, entropy, 0.0).float()}
    if c["top"]:
        ids = logits.sort(dim=-1, descending=True, stable=True)[1]
        ids = ids[:, :c["top"]]
        best = (d.gather(1, ids).double() - log_total).float()
        r["top_logprobs"] = torch.where(keep[:, None], best, -math.inf)
        r["top_ids"] = torch.where(keep[:, None], ids, -1)
    if "d_logprob" in s:
        up = s["d_logprob"][:, None]
        if "d_top" in s:
            up = up + s["d_top"].sum(-1, keepdim=True)
        if "d_entropy" in s:
            lean = (entropy[:, None] - log_total).float()   # l + H = d + lean
            up = up + s["d_entropy"][:, None] * (d + lean)
        grad = e * (1.0 / total).float() * -up
        grad.scatter_add_(1, at, s["d_logprob"][:, None])
        if "d_top" in s:
            grad.scatter_add_(1, ids, s["d_top"])
        grad = torch.where(keep[:, None], grad / c["temperature"], 0.0)
        r["dlogits"] = grad.to(logits.dtype)
    return r


def _plain_distill(s):
    c, logits, ids = s["case"], s["logits"], s["top_ids"]
    rows, width = logits.shape
    present = ids >= 0
    at = torch.where(present, ids, width)     # absent ones go to a last column
    t = torch.where(present, s["top_logprobs"], -math.inf).double()
    if c["tail"]:
        q = t.exp()
        rest = (1.0 - q.sum(-1)).clamp(min=0.0)
    else:
        m = t.amax(-1, keepdim=True)
        q = (t - torch.where(m == -math.inf, 0.0, m)).exp()
        q = q / q.sum(-1, keepdim=True).clamp(min=1e-300)
        rest = torch.zeros(rows, dtype=torch.double, device=q.device)
    live = present.any(-1)
    d, e, total = _plain_softmax(logits, c["temperature"])
    l_at = d.gather(1, at.clamp(max=width - 1)).double() - total.log()
    loss = torch.where(q > 0, q * (q.log() - l_at), 0.0).sum(-1)
    if c["tail"]:
        named = torch.zeros(rows, width + 1, dtype=torch.bool,
                            device=q.device)
        named = named.scatter_(1, at, True)[:, :width]
        out = torch.where(named, 0.0, e).sum(-1, dtype=torch.double) \
            / total[:, 0]
        has = (rest > 0) & (out > 0)
        loss = loss + torch.where(has, rest * (rest.log() - out.log()), 0.0)
    scale = c["temperature"]
    r = {"loss": torch.where(live, loss * (scale * scale), 0.0).float()}
    if "d_loss" in s:
        share = q.sum(-1)[:, None]
        if c["tail"]:
            share = share + torch.where(has, rest, 0.0)[:, None]
            shift = torch.where(has, rest / out, 0.0)[:, None]
            factor = torch.where(named, share.float(),
                                 (share - shift).float())
        else:
            factor = share.float()
        grad = e * (1.0 / total).float() * factor
        taught = torch.zeros(rows, width + 1, device=q.device)
        grad = grad - taught.scatter_add_(1, at, q.float())[:, :width]
        grad = grad * (s["d_loss"] * scale)[:, None]
        r["dlogits"] = torch.where(live[:, None], grad, 0.0).to(logits.dtype)
    return r


# --------------------------------------------------- the package's entry points
def _own_norm(s):
    from dear_pytorch_amd.ops.fused_ln import layer_norm
    y = layer_norm(s["x"], s["weight"], s["bias"], _EPS,
                   residual=s.get("residual"))
    r = {"y": y}
    if "dy" in s:
        names = [k for k in ("x", "residual", "weight", "bias") if k in s]
        got = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
        r.update({"d" + k: g for k, g in zip(names, got)})
    return r


def _own_logprobs(s):
    from dear_pytorch_amd.ops.token_loss import token_logprobs
    c = s["case"]
    t = token_logprobs(s["logits"], s["tokens"], top=c["top"],
                       temperature=c["temperature"])
    r = {"logprob": t.logprob, "entropy": t.entropy}
    if c["top"]:
        r["top_logprobs"], r["top_ids"] = t.top_logprobs, t.top_ids
    if "d_logprob" in s:
        outs, ups = [t.logprob], [s["d_logprob"]]
        if "d_entropy" in s:
            outs.append(t.entropy)
            ups.append(s["d_entropy"])
        if "d_top" in s:
            outs.append(t.top_logprobs)
            ups.append(s["d_top"])
        r["dlogits"], = torch.autograd.grad(outs, [s["logits"]], ups)
    return r


def _own_distill(s):
    from dear_pytorch_amd.ops.token_loss import topk_distill_loss
    c = s["case"]
    loss = topk_distill_loss(s["logits"], s["top_ids"], s["top_logprobs"],
                             temperature=c["temperature"], tail=c["tail"])
    r = {"loss": loss}
    if "d_loss" in s:
        r["dlogits"], = torch.autograd.grad(loss, [s["logits"]], s["d_loss"])
    return r


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "logprobs": _own_logprobs,
                "distill": _own_distill}[op](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "logprobs": _plain_logprobs,
                "distill": _plain_distill}[op](state)


# ------------------------------------------------------------------- the work
def work(case):
    rows, width, grad = case["rows"], case["width"], case["grad"]
    size = 4 if case["dtype"] == "fp32" else 2
    n = rows * width
    if case["op"] == "norm":
        wide = 4 if case["dtype"] in ("fp32", "amp") else 2
        out = wide if case["residual"] else size
        total = n * size + n * out + 2 * width * wide      # x, y, weight, bias
        if case["residual"]:
            total += n * wide
        if grad:
            total += n * out + n * size + 2 * width * wide  # dy, dx, dw, db
            if case["residual"] and wide != size:
                total += n * wide                           # dresidual
        return {"bytes": total, "flops": n * (20 if grad else 8)}
    read = n * case["labelled"]
    total = read * size + rows * (8 + 12 * case["top"] + 8)
    if grad:
        total += n * size + 4 * rows
    return {"bytes": int(total), "flops": int(read * (10 if grad else 5))}


# ------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    leaf = {k: v.detach().double().requires_grad_(case["grad"])
            for k, v in s.items()
            if k in ("x", "residual", "weight", "bias", "logits")}
    if case["op"] == "norm":
        z = leaf["x"] + leaf["residual"] if case["residual"] else leaf["x"]
        var, mean = torch.var_mean(z, dim=-1, correction=0, keepdim=True)
        y = (z - mean) / torch.sqrt(var + _EPS) * leaf["weight"] \
            + leaf["bias"]
        r = {"y": y.detach()}
        if case["grad"]:
            got = torch.autograd.grad(y, list(leaf.values()),
                                      s["dy"].double())
            r.update({"d" + k: g for k, g in zip(leaf, got)})
        return r
    logp = torch.log_softmax(leaf["logits"] / case["temperature"], dim=-1)
    rows, width = logp.shape
    if case["op"] == "logprobs":
        keep = s["tokens"] >= 0
        picked = logp[torch.arange(rows, device=_DEVICE),
                      s["tokens"].clamp(min=0)]
        logprob = torch.where(keep, picked, 0.0)
        entropy = torch.where(keep, -(logp.exp() * logp).sum(-1), 0.0)
        outs = {"logprob": logprob, "entropy": entropy}
        if case["top"]:
            # the gathered values do not depend on which of two equals is taken
            best = logp.topk(case["top"], dim=-1)[0]
            outs["top_logprobs"] = torch.where(keep[:, None], best, -math.inf)
        r = {k: v.detach() for k, v in outs.items()}
        if case["top"]:
            r["top_ids"] = None
        if case["grad"]:
            total = (logprob * s["d_logprob"].double()).sum()
            if case["entropy_grad"]:
                total = total + (entropy * s["d_entropy"].double()).sum()
                if case["top"]:
                    # which of two equals is taken matters to the gradient
                    ids = s["logits"].detach().sort(
                        dim=-1, descending=True, stable=True)[1]
                    best = logp.gather(1, ids[:, :case["top"]])
                    total = total + (best * s["d_top"].double()
                                     * keep[:, None]).sum()
            r["dlogits"], = torch.autograd.grad(total, [leaf["logits"]])
        return r
    # distillation: the Kullback-Leibler divergence of two distributions over
    # the named tokens (and one bucket for all others)
    ids, present = s["top_ids"].clamp(min=0), s["top_ids"] >= 0
    live = present.any(-1)
    teacher = s["top_logprobs"].double().masked_fill(~present, -math.inf)
    teacher = teacher.masked_fill(~live[:, None], 0.0)
    if not case["tail"]:
        teacher = torch.log_softmax(teacher, dim=-1)
    q = teacher.exp()
    gap = torch.where(q > 0, teacher - logp.gather(1, ids), 0.0)
    loss = (q * gap).sum(-1)
    if case["tail"]:
        rest = (1.0 - q.sum(-1)).clamp(min=0.0)
        off = torch.zeros(rows, width, dtype=torch.double, device=_DEVICE)
        off = off.scatter_add_(1, ids, present.double()) > 0
        out = logp.masked_fill(off, -math.inf).logsumexp(-1)
        some = (rest > 0) & live & torch.isfinite(out)
        loss = loss + torch.where(some, rest * (
            torch.where(some, rest, 1.0).log() - out), 0.0)
    loss = torch.where(live, loss * case["temperature"] ** 2, 0.0)
    r = {"loss": loss.detach()}
    if case["grad"]:
        r["dlogits"], = torch.autograd.grad(loss, [leaf["logits"]],
                                            s["d_loss"].double())
    return r
