"""Residual add + layer norm against the formula in float64: the CPU
composition, the HIP kernels (gpu-marked), and what is refused.

Bounds: u is half a step of float32 (2^-24). A float32 sum of n terms in a
chain is off by at most n u times the sum of their magnitudes, a tree by its
depth; a thread adds at most H / 64 + 64 elements before the tree, so `chain`
covers both. With M the largest |z| of the row:
    mean, z - mean:  off by at most u (chain + 2) M
    rstd:            relatively by u (chain + 6) + that times rstd
    n:               by E = u ((chain + 4) M rstd + (chain + 12) |n|)
and each later product or sum adds one u of its result. A 16-bit result adds
half a step of its type, and float16 half of its smallest step (2^-25)."""
import pytest
import torch
import torch.nn as nn

from dear_pytorch_amd.ops.fused_ln import FusedLayerNorm, layer_norm

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8,
        torch.float16: 2.0 ** -11}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def rounded(err, value, dtype):
    """The bound `err` of a float32 value, after its rounding to dtype."""
    tiny = 2.0 ** -25 if dtype == F16 else 2.0 ** -134
    return err + HALF[dtype] * (value.abs() + err) + tiny


def exact(x, w, b, eps, res, dy):
    """Value, gradients and their bounds in float64, from the formulas."""
    z = x.double()
    if res is not None:
        z = z + res.double()
    H = z.size(-1)
    z2 = z.reshape(-1, H)
    chain = H / 64 + 64 + 10
    mean = z2.mean(-1, keepdim=True)
    d = z2 - mean
    rstd = 1.0 / (d.square().mean(-1, keepdim=True) + eps).sqrt()
    n = d * rstd
    wd = torch.ones(H, dtype=torch.double, device=x.device) if w is None \
        else w.double()
    y = n * wd + (0 if b is None else b.double())
    big = z2.abs().amax(-1, keepdim=True)
    E = U * ((chain + 4) * big * rstd + (chain + 12) * n.abs())
    y_err = E * wd.abs() + 2 * U * ((n * wd).abs() + y.abs())
    out = {"y": (y.view_as(z), y_err.view_as(z))}
    if dy is None:
        return out
    g0 = dy.double().reshape(-1, H)
    g = g0 * wd
    mg, mgn = g.mean(-1, keepdim=True), (g * n).mean(-1, keepdim=True)
    dz = rstd * (g - mg - n * mgn)
    ag, agn = g.abs().mean(-1, keepdim=True), (g * n).abs().mean(-1, True)
    Emax = E.amax(-1, keepdim=True)
    rel = U * (chain + 6) + U * (chain + 2) * big * rstd
    dz_err = rstd * (U * (4 * g.abs() + (chain + 6) * ag
                          + n.abs() * (chain + 8) * agn)
                     + E * mgn.abs() + n.abs() * ag * Emax) \
        + dz.abs() * (rel + 4 * U)
    out["dz"] = (dz.view_as(z), dz_err.view_as(z))
    rows = z2.size(0)
    out["dw"] = ((g0 * n).sum(0), (g0.abs() * (E + 2 * U * n.abs())).sum(0)
                 + U * (rows + 2) * (g0 * n).abs().sum(0))
    out["db"] = (g0.sum(0), U * (rows + 2) * g0.abs().sum(0))
    return out


def check(got, want, what):
    value, err = want
    bound = rounded(err, value, got.dtype)
    off = (got.double() - value).abs()
    worst = (off / bound.clamp(min=1e-300)).max().item() if off.numel() else 0
    assert got.shape == value.shape and worst <= 1.0, (what, worst)


def run(x, w, b, eps, res, dy=None):
    leaves = {k: t.detach().requires_grad_(True) for k, t in
              (("x", x), ("res", res), ("w", w), ("b", b)) if t is not None}
    y = layer_norm(leaves["x"], leaves.get("w"), leaves.get("b"), eps,
                   residual=leaves.get("res"))
    grads = torch.autograd.grad(y, list(leaves.values()), dy)
    return y.detach(), dict(zip(leaves, grads))


def compare(x, w, b, eps, res, dy):
    y, g = run(x, w, b, eps, res, dy)
    want = exact(x, w, b, eps, res, dy)
    wide = x.dtype if res is None else torch.promote_types(x.dtype, res.dtype)
    assert y.dtype == wide and y.is_contiguous()
    check(y, want["y"], "y")
    for name, key in (("x", "dz"), ("res", "dz"), ("w", "dw"), ("b", "db")):
        if name in g:
            src = {"x": x, "res": res, "w": w, "b": b}[name]
            assert g[name].dtype == src.dtype
            check(g[name], want[key], name)
    # no graph is kept where nothing asks for one; the value is the same
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps, residual=res), y)


def make(rows, H, tx, tr, tw, dev, affine="wb", seed=0):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)
    wide = tx if tr is None else torch.promote_types(tx, tr)
    x = (rand(rows, H) * 2 + rand(rows, 1)).to(tx)
    res = None if tr is None else rand(rows, H).to(tr)
    w = (1 + 0.2 * rand(H)).to(tw) if "w" in affine else None
    b = (0.2 * rand(H)).to(tw) if "b" in affine else None
    dy = rand(rows, H).to(wide)
    return [None if t is None else t.to(dev) for t in (x, w, b, res, dy)]


# ------------------------------------------------------------------- on CPU
@pytest.mark.parametrize("tx,tr,tw", [
    (F32, None, F32), (F32, F32, F32), (BF16, F32, F32), (F32, F16, F32),
    (BF16, BF16, BF16)])
@pytest.mark.parametrize("rows,H", [(3, 1), (5, 77), (0, 8)])
def test_cpu_composition(rows, H, tx, tr, tw):
    x, w, b, res, dy = make(rows, H, tx, tr, tw, "cpu")
    compare(x, w, b, 1e-5, res, dy)


def test_cpu_equals_torch_in_fp32():
    x, w, b, res, _ = make(9, 40, F32, F32, F32, "cpu")
    want = nn.functional.layer_norm(x + res, (40,), w, b, 1e-5)
    assert torch.equal(layer_norm(x, w, b, 1e-5, residual=res), want)


def test_gradients_against_differences():
    gen = torch.Generator().manual_seed(5)
    args = [torch.randn(4, 6, generator=gen, dtype=torch.double,
                        requires_grad=True),
            *(torch.randn(6, generator=gen, dtype=torch.double)
              .requires_grad_(True) for _ in range(2)),
            torch.randn(4, 6, generator=gen, dtype=torch.double,
                        requires_grad=True)]
    assert torch.autograd.gradcheck(
        lambda x, w, b, r: layer_norm(x, w, b, 1e-5, residual=r), args)


def test_module_is_state_dict_compatible():
    fused, plain = FusedLayerNorm(16, eps=1e-12), nn.LayerNorm(16, eps=1e-12)
    fused.load_state_dict(plain.state_dict())
    plain.load_state_dict(fused.state_dict())
    x = torch.randn(3, 16)
    assert torch.equal(fused(x), plain(x))
    assert torch.equal(fused(x, residual=x), plain(x + x))
    assert FusedLayerNorm(4, elementwise_affine=False)(torch.ones(2, 4)) \
        .abs().max() == 0
    assert FusedLayerNorm(4, bias=False).bias is None


def bad_calls(dev="cpu"):
    x = torch.zeros(2, 8, device=dev)
    h, b16 = x.half(), x.bfloat16()
    w = torch.ones(8, device=dev)
    return [
        (ValueError, (torch.zeros((), device=dev), None, None, None)),
        (ValueError, (torch.zeros(3, 0, device=dev), None, None, None)),
        (TypeError, (x.int(), None, None, None)),
        (TypeError, (x, None, None, x.int())),
        (ValueError, (x, None, None, x[:1])),
        (ValueError, (x, None, None, torch.zeros(8, device=dev))),
        (TypeError, (h, None, None, b16)),
        (ValueError, (x, w[:7], None, None)),
        (ValueError, (x, w.view(1, 8), None, None)),
        (ValueError, (x, torch.ones(16, device=dev)[::2], None, None)),
        (TypeError, (x, w.half(), None, None)),
        (TypeError, (b16, w.half(), None, None)),
        (TypeError, (h, w.half(), w, None)),
    ]


@pytest.mark.parametrize("i", range(len(bad_calls())))
def test_refusals(i):
    err, (x, w, b, r) = bad_calls()[i]
    with pytest.raises(err):
        layer_norm(x, w, b, 1e-5, residual=r)
    kernels = pytest.importorskip("dear_pytorch_amd._kernels")
    with pytest.raises(err):
        kernels.layer_norm(x, w, b, 1e-5, r)


def test_refusals_of_module_and_eps():
    with pytest.raises(ValueError):
        FusedLayerNorm((4, 4))
    with pytest.raises(ValueError):
        FusedLayerNorm(4)(torch.zeros(2, 5))
    for eps in (-1e-5, float("nan")):
        with pytest.raises(ValueError):
            layer_norm(torch.zeros(2, 4), eps=eps)


# ------------------------------------------------------------------ on a GPU
TYPES = [(F32, None, F32), (BF16, None, BF16), (F16, None, F32),
         (F32, F32, F32), (BF16, BF16, F32), (F16, F16, F16),
         (BF16, F32, F32), (F32, F16, F32)]


@pytest.mark.gpu
@pytest.mark.parametrize("tx,tr,tw", TYPES)
@pytest.mark.parametrize("rows,H", [
    (1, 1), (3, 2), (70, 7), (1, 768), (130, 63), (65, 64), (9, 65),
    (257, 255), (33, 768), (517, 1011), (31, 1024), (6, 2047), (5, 4099),
    (3, 8192), (2, 20011), (2, 70001)])
def test_gpu_against_float64(rows, H, tx, tr, tw):
    x, w, b, res, dy = make(rows, H, tx, tr, tw, "cuda", seed=rows + H)
    compare(x, w, b, 1e-5, res, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("affine", ["", "w", "b"])
def test_gpu_without_weight_or_bias(affine):
    for tw in (F32, BF16):
        x, w, b, res, dy = make(21, 96, BF16, BF16, tw, "cuda", affine)
        compare(x, w, b, 1e-12, res, dy)


@pytest.mark.gpu
def test_gpu_many_rows_weight_gradient():
    x, w, b, res, dy = make(20000, 40, F32, F32, F32, "cuda")
    compare(x, w, b, 1e-5, res, dy)


@pytest.mark.gpu
def test_gpu_no_rows():
    x, w, b, res, dy = make(0, 24, F32, F32, F32, "cuda")
    y, g = run(x, w, b, 1e-5, res, dy)
    assert y.shape == (0, 24) and g["x"].shape == (0, 24)
    assert g["w"].abs().sum() == 0 and g["b"].abs().sum() == 0


@pytest.mark.gpu
def test_gpu_strides():
    x, w, b, res, dy = make(40, 200, F32, F32, F32, "cuda")
    cut = slice(3, 180)                      # rows that start off a boundary
    compare(x[:, cut], w[cut], b[cut].contiguous(), 1e-5, res[:, cut],
            dy[:, cut])
    compare(x[::3], w, b, 1e-5, res[::3], dy[:14])            # a row stride
    compare(x.t().contiguous().t(), w, b, 1e-5, res, dy)      # columns first
    compare(x, w, b, 1e-5, res[:1].expand(40, 200), dy)       # a stride of 0
    compare(x, w, b, 1e-5, res, dy[:1, :1].expand(40, 200))
    compare(x.view(5, 8, 200).transpose(0, 1), w, b, 1e-5,
            res.view(8, 5, 200), dy.view(8, 5, 200))
    compare(x[7], w, b, 1e-5, res[7], dy[7])                  # one axis
    v = x.half()[:, 1:94]                                     # odd halves
    compare(v, None, None, 1e-5, None, dy.half()[:, 1:94])


@pytest.mark.gpu
def test_gpu_only_some_gradients():
    x, w, b, res, dy = make(37, 130, BF16, F32, F32, "cuda")
    _, full = run(x, w, b, 1e-5, res, dy)
    leaves = {"x": x, "w": w, "b": b, "res": res}
    for names in (["x"], ["res"], ["w"], ["b"], ["x", "b"]):
        t = {k: v.detach().requires_grad_(k in names)
             for k, v in leaves.items()}
        y = layer_norm(t["x"], t["w"], t["b"], 1e-5, residual=t["res"])
        got = torch.autograd.grad(y, [t[k] for k in names], dy)
        for k, v in zip(names, got):
            assert torch.equal(v, full[k]), (names, k)


@pytest.mark.gpu
def test_gpu_residual_is_x():
    x, w, b, _, dy = make(11, 50, F32, None, F32, "cuda")
    leaf = x.requires_grad_(True)
    y = layer_norm(leaf, w, b, 1e-5, residual=leaf)
    g, = torch.autograd.grad(y, leaf, dy)
    want = exact(x.detach(), w, b, 1e-5, x.detach(), dy)
    value, err = want["dz"]
    check(g, (2 * value, 2 * rounded(err, value, F32)), "x twice")


@pytest.mark.gpu
def test_gpu_offset_far_larger_than_the_spread():
    # the statistics see the spread, not the square of the offset
    x, w, b, _, dy = make(8, 768, F32, None, F32, "cuda")
    compare(x * 1e-2 + 100.0, w, b, 1e-12, None, dy)


@pytest.mark.gpu
def test_gpu_constant_rows_and_eps():
    x = torch.full((4, 256), 3.0, device="cuda")
    w = torch.ones(256, device="cuda")
    assert layer_norm(x, w, w, 1e-12).eq(1.0).all()
    # a row of one element: its variance is zero whatever it holds
    assert layer_norm(x[:, :1], None, None, 1e-5).eq(0.0).all()


@pytest.mark.gpu
def test_gpu_bad_rows_stay_alone():
    x, w, b, res, dy = make(12, 300, F32, F32, F32, "cuda")
    good = run(x, w, b, 1e-5, res, dy)
    bad = x.clone()
    bad[3, 7], bad[5, 0], bad[9, 299] = float("nan"), float("inf"), \
        -float("inf")
    y, g = run(bad, w, b, 1e-5, res, dy)
    rows = [3, 5, 9]
    keep = [i for i in range(12) if i not in rows]
    assert torch.isnan(y[rows]).all() and torch.isnan(g["x"][rows]).all()
    assert torch.equal(y[keep], good[0][keep])
    assert torch.equal(g["x"][keep], good[1]["x"][keep])


@pytest.mark.gpu
def test_gpu_same_call_same_bits():
    x, w, b, res, dy = make(3000, 1011, F16, None, F32, "cuda")
    a, ga = run(x, w, b, 1e-5, res, dy)
    for _ in range(3):
        c, gc = run(x, w, b, 1e-5, res, dy)
        assert torch.equal(a, c) and all(torch.equal(ga[k], gc[k])
                                         for k in ga)


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    H, rows = 1024, (1 << 21) + 5            # over 2^31 elements
    x = torch.empty(rows, H, dtype=BF16, device="cuda")
    x[:4], x[-4:] = torch.randn(2, 4, H, device="cuda").to(BF16)
    x[4:-4] = x[0]
    w = torch.ones(H, device="cuda")
    y = layer_norm(x, w, None, 1e-5)
    for part in (slice(0, 4), slice(rows - 4, rows)):
        check(y[part], exact(x[part], w, None, 1e-5, None, None)["y"], part)
    del y
    leaf = x.requires_grad_(True)
    y = layer_norm(leaf, w, None, 1e-5)
    dy = torch.randn(1, H, device="cuda").to(BF16).expand(rows, H)
    g, = torch.autograd.grad(y, leaf, dy)
    part = slice(rows - 4, rows)
    check(g[part], exact(x.detach()[part], w, None, 1e-5, None,
                         dy[part])["dz"], "dz")


@pytest.mark.gpu
def test_gpu_streams_and_graph():
    x, w, b, res, dy = make(64, 768, F32, F32, F32, "cuda")
    want, gwant = run(x, w, b, 1e-5, res, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, g = run(x, w, b, 1e-5, res, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want) and torch.equal(g["w"], gwant["w"])
    # captured forward and backward, replayed on new inputs between eager work
    sx, sdy = x.clone(), dy.clone()
    graphs = []
    for _ in range(2):                       # two graphs, each its workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(sx, w, b, 1e-5, res, sdy)
        graphs.append((graph, out))
    for i in range(4):
        sx.copy_(torch.roll(x, i, 0))
        sdy.copy_(torch.roll(dy, i, 1))
        ye, ge = run(sx, w, b, 1e-5, res, sdy)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, (yg, gg) in graphs:
            assert torch.equal(yg, ye)
            assert all(torch.equal(gg[k], ge[k]) for k in ge), i


@pytest.mark.gpu
def test_gpu_capture_beside_a_live_eager_graph_is_refused():
    x, w, b, _, dy = make(8, 64, F32, F32, F32, "cuda")
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    alive = layer_norm(*leaves)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer_norm(*leaves)
        with pytest.raises(RuntimeError, match="alive"):
            torch.autograd.grad(y, leaves, dy)
    want = torch.autograd.grad(alive, leaves, dy)
    del alive, y
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, v) for g, v in zip(got, want))


@pytest.mark.gpu
def test_gpu_second_derivative_is_refused():
    x, w, b, _, _ = make(4, 16, F32, None, F32, "cuda")
    x.requires_grad_(True)
    g, = torch.autograd.grad(layer_norm(x, w, b).square().sum(), x,
                             create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()


@pytest.mark.gpu
def test_gpu_refuses_what_the_kernel_lacks():
    x = torch.zeros(2, 8, device="cuda")
    with pytest.raises(TypeError):
        layer_norm(x.double())
    with pytest.raises(ValueError):
        layer_norm(x, torch.ones(8))
    with pytest.raises(ValueError):
        layer_norm(x, residual=torch.zeros(2, 8))


@pytest.mark.gpu
def test_gpu_module_in_training():
    x, _, _, r, dy = make(35, 96, F32, F32, F32, "cuda")
    shape = (5, 7, 96)
    x, r, dy = x.view(shape), r.view(shape), dy.view(shape)
    fused = FusedLayerNorm(96, eps=1e-12).cuda()
    fused(x, residual=r).backward(dy)
    want = exact(x, fused.weight.detach(), fused.bias.detach(), 1e-12, r, dy)
    check(fused.weight.grad, want["dw"], "weight")
    check(fused.bias.grad, want["db"], "bias")
