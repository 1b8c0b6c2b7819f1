"""Layer norm of rows whose mean is far larger than their spread, or that have
no spread at all, against the formula in float64.

Without a residual z is x itself, and then no error goes by the size of z:
u is half a step of float32 (2^-24), `chain` the additions behind a sum (a
thread's, then a tree, as in test_fused_ln), s the row's standard deviation.
Where the mean's first rounding is an eighth of s at most, a second sum over
z - mean takes it out: what is left of the mean is off by u chain mean|z - mean|
<= 1.2 u chain s, and so is n = (z - mean) rstd by
    E = u (chain + 12) (1.5 + |n|).
Otherwise the mean is rounded again and the distances to it are exact. Counted
in steps of z they are whole numbers k with |mean k| <= 1/2, so mean |k| <=
mean k^2 <= 2 (mean k^2 - (mean k)^2), and mean|z - mean| <= 1.5 s: the same E.
Equal elements leave nothing at all."""
import pytest
import torch

from dear_pytorch_amd.ops.fused_ln import layer_norm
from test_fused_ln import BF16, F16, F32, HALF, U, check, run

WIDTHS = [5, 63, 768, 1011, 1024, 4099, 8192, 16384, 20011]


def exact(x, w, b, eps, dy):
    z = x.double()
    H = z.size(-1)
    chain = H / 64 + 64 + 10
    d = z - z.mean(-1, keepdim=True)
    d = d - d.mean(-1, keepdim=True)
    rstd = 1.0 / (d.square().mean(-1, keepdim=True) + eps).sqrt()
    n = d * rstd
    E = U * (chain + 12) * (1.5 * (d != 0).any(-1, keepdim=True) + n.abs())
    w, b, g0 = w.double(), b.double(), dy.double()
    y = n * w + b
    out = {"y": (y, E * w.abs() + 2 * U * ((n * w).abs() + y.abs()))}
    g = g0 * w
    mg, mgn = g.mean(-1, keepdim=True), (g * n).mean(-1, keepdim=True)
    ag, agn = g.abs().mean(-1, keepdim=True), (g * n).abs().mean(-1, True)
    dz = rstd * (g - mg - n * mgn)
    dz_err = rstd * (U * (4 * g.abs() + (chain + 6) * ag
                          + n.abs() * (chain + 8) * agn)
                     + E * mgn.abs()
                     + n.abs() * (g.abs() * E).mean(-1, keepdim=True)) \
        + dz.abs() * U * (2 * chain + 16)
    out["x"] = (dz, dz_err)
    rows = z.size(0)
    out["w"] = ((g0 * n).sum(0), (g0.abs() * (E + 2 * U * n.abs())).sum(0)
                + U * (rows + 2) * (g0 * n).abs().sum(0))
    return out


def affine(rows, H, dtype):
    gen = torch.Generator().manual_seed(rows + H)
    w = (1 + 0.2 * torch.randn(H, generator=gen)).to(F32)
    b = (0.2 * torch.randn(H, generator=gen)).to(F32)
    dy = torch.randn(rows, H, generator=gen).to(dtype)
    return w.cuda(), b.cuda(), dy.cuda()


def check_range(got, want, what):
    """check, where a number past its type's range is the infinity that it
    rounds to: rstd is up to 1e6 here, and float16 ends at 65504."""
    value, err = want
    past = torch.isinf(got)
    most = torch.finfo(got.dtype).max
    assert (value.abs() + err)[past].ge(most).all(), what
    assert torch.equal(got[past] > 0, value[past] > 0), what
    check(torch.where(past, 0.0, got), (torch.where(past, 0.0, value), err),
          what)


def compare(x, eps):
    w, b, dy = affine(*x.shape, x.dtype)
    x = x.cuda()
    y, g = run(x, w, b, eps, None, dy)
    want = exact(x, w, b, eps, dy)
    check(y, want["y"], "y")
    for k in ("x", "w"):
        check_range(g[k], want[k], k)
    return y, b, g


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("H", WIDTHS)
def test_gpu_equal_elements_are_their_mean(H, dtype):
    values = torch.tensor([1000.1, 0.1, 3.0, -19.7, 1.0 / 3, 1e-3, -33333.3,
                           5e-5])
    x = values[:, None].to(dtype).repeat(1, H)
    y, b, g = compare(x, 1e-12)
    assert torch.equal(y, b.to(dtype).expand_as(y))
    assert (g["w"] == 0).all()
    # a branch and a residual whose sums are equal
    r = torch.full_like(x, 0.0).float().cuda() + 7.7
    y = layer_norm(x.cuda(), None, None, 1e-12, residual=r)
    assert (y == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [1e-12, 1e-5])
@pytest.mark.parametrize("H", WIDTHS)
def test_gpu_spread_of_a_few_steps(H, eps):
    """Elements that differ by single steps of float32, one of them only, and
    the other way round."""
    gen = torch.Generator().manual_seed(H)
    c = torch.tensor([1000.1, 0.1, 19.7, 65535.9])[:, None]
    step = torch.nextafter(c, torch.tensor(1e9)) - c
    some = torch.randint(-2, 3, (4, H), generator=gen)
    one = torch.zeros(4, H)
    one[:, H // 2] = 1
    rows = [c + step * some, c + step * one, -(c - step * one)]
    compare(torch.cat(rows).contiguous(), eps)


@pytest.mark.gpu
@pytest.mark.parametrize("H", WIDTHS)
def test_gpu_offsets_of_every_size(H):
    gen = torch.Generator().manual_seed(H + 1)
    offset = 2.0 ** torch.arange(0, 24)[:, None]
    x = torch.randn(24, H, generator=gen) + offset * 1.37
    compare(x, 1e-12)


@pytest.mark.gpu
def test_gpu_rows_of_both_kinds_share_a_wave():
    """Rows of 16 threads: some lanes of a wave take the second round, the
    others do not."""
    gen = torch.Generator().manual_seed(8)
    for H in (7, 64, 100):
        x = torch.randn(37, H, generator=gen)
        x[::3] = x[::3, :1]                      # no spread
        x[1::4] += 1000.1
        compare(x, 1e-12)


@pytest.mark.gpu
def test_gpu_wider_than_a_launch_of_its_columns():
    """Over 2^27 columns: their sums of 1024 threads for 64 of them would be
    more threads than a launch holds."""
    H = (1 << 27) + 70
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, dy = torch.randn(2, 1, H, generator=gen, device="cuda")
    w, b = torch.ones(H, device="cuda"), torch.zeros(H, device="cuda")
    _, g = run(x, w, b, 1e-5, None, dy)
    assert torch.equal(g["b"], dy[0])
    z = x[0].double()
    n = (z - z.mean()) / (z.var(correction=0) + 1e-5).sqrt()
    # n rounds in a difference of three, a root, a quotient and a product
    err = 8 * U * (n.abs() + 1)
    check(g["w"], (dy[0] * n, dy[0].abs().double() * err), "w")


@pytest.mark.gpu
@pytest.mark.parametrize("H", [20011, 3000001])
def test_gpu_long_rows_sum_without_drift(H):
    """A constant upstream gradient, which each thread adds up in one chain: the
    gradient of x is what the sums leave of it, and these are float64 here. The
    products round once each, and g - mean g - n mean(g n) twice more."""
    gen = torch.Generator().manual_seed(H)
    x = torch.randn(2, H, generator=gen).cuda()
    dy = torch.full_like(x, 0.1)
    dy[1, ::2] = 0.3
    _, g = run(x, None, None, 1e-5, None, dy)
    z, up = x.double(), dy.double()
    d = z - z.mean(-1, keepdim=True)
    rstd = 1.0 / (d.square().mean(-1, keepdim=True) + 1e-5).sqrt()
    n = d * rstd
    mgn = (up * n).mean(-1, keepdim=True)
    dz = rstd * (up - up.mean(-1, keepdim=True) - n * mgn)
    # n is off by 8 u (|n| + 1); the mean of g n by as much of mean |g n|
    off = (up.abs() * 8 * U * (n.abs() + 1)).mean(-1, keepdim=True)
    err = rstd * (4 * U * up.abs() + off * n.abs()
                  + 8 * U * (n.abs() + 1) * mgn.abs()) + 6 * U * dz.abs()
    check(g["x"], (dz, err), "x")
