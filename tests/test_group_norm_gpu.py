"""Group norm with activation (csrc/group_norm.hip) against its definition in 64 bits, forward and backward.

Tolerances, element by element (u = half a step of the tensor's type, f = 2^-20 for the fp32 arithmetic in between: statistics of up
to 2^20 values summed in runs of at most 2^4 terms in a row, a handful of operations and two hardware transcendentals each good to
2 units of 2^-23):
  y   u |y| + f (|n gamma| + |beta| + |gamma| m), m = |mean| rstd: a mean off by f of the spread or of itself shifts n
  dx  u |dx| + f rstd (|dz gamma| + avg |dz gamma| + |n| avg |dz gamma n|), times what m adds to n
  sums  f times the sum of the magnitudes
"""
import pytest
import torch

from oracle import attention as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def inputs(seed, shape, dtype, mean=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    C = shape[-1]
    return (r(*shape) * (0.5 + r(C).abs()) + mean * r(C)).to(dtype), 1 + 0.3 * r(C), 0.3 * r(C), r(*shape).to(dtype)


def run(x, gamma, beta, dy, groups, act, eps=1e-5, slope=0.2):
    from rgbd_gan_amd import functional as Fn
    leaves = [t.detach().requires_grad_(True) for t in (x, gamma, beta)]
    y = Fn.group_norm(*leaves, groups, eps, act, slope)
    return (y.detach(), *torch.autograd.grad(y, leaves, dy))


def check(x, gamma, beta, dy, groups, act, eps=1e-5, slope=0.2):
    got = run(x, gamma, beta, dy, groups, act, eps, slope)
    leaves = [t.detach().to(F64).requires_grad_(True) for t in (x, gamma, beta)]
    want_y = ref.group_norm(*leaves, groups, eps, act, slope)
    want = (want_y.detach(), *torch.autograd.grad(want_y, leaves, dy.to(F64)))
    u, f = {BF16: 2.0 ** -8, F32: 2.0 ** -24}[x.dtype], 2.0 ** -20
    B, C = x.shape[0], x.shape[-1]
    xd, gd, bd, dyd = (t.detach().to(F64) for t in (x, gamma, beta, dy))
    v = xd.reshape(B, -1, groups, C // groups)
    mean = v.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((v - mean) ** 2).mean(dim=(1, 3), keepdim=True) + eps)
    wide = lambda t: (t + torch.zeros_like(v)).reshape(x.shape)
    n, m, rs = wide((v - mean) * rstd), wide(mean.abs() * rstd), wide(rstd)
    z = n * gd + bd
    d = torch.ones_like(z)
    if act == "silu":
        s = torch.sigmoid(z)
        d = s * (1 + z * (1 - s))
    elif act == "lrelu":
        d = torch.where(z > 0, 1.0, slope).to(F64)
    size = 1.1 if act == "silu" else max(1.0, abs(slope))
    ez = f * ((n * gd).abs() + bd.abs() + gd.abs() * (1 + m))                       # what z may be off by
    tol_y = u * want[0].abs() + size * ez + 1e-30
    # act' moves with z: by at most 1/2 of its error (SiLU); a leaky ReLU's jumps where |z| is below the error
    ed = 0.5 * ez + f if act == "silu" else ((z.abs() <= ez).to(F64) * abs(1 - slope) if act == "lrelu" else 0 * z)
    dz, edz = dyd * d, dyd.abs() * (ed + f * d.abs())
    en = f * (n.abs() + 1 + m)
    avg = lambda t: wide(t.reshape(v.shape).mean(dim=(1, 3), keepdim=True))
    dn, edn = dz * gd, edz * gd.abs()
    mag = dn.abs() + avg(dn.abs()) + n.abs() * avg((dn * n).abs())
    tol_dx = (u * want[1].abs() + rs * (f * mag + edn + avg(edn) + n.abs() * avg(edn * n.abs() + dn.abs() * en) + en * avg((dn * n).abs()))
              + 1e-30)
    total = lambda t: t.reshape(-1, C).sum(0)
    tol_g = total(f * (dz * n).abs() + edz * n.abs() + dz.abs() * en) + 1e-30
    tol_b = total(f * dz.abs() + edz) + 1e-30
    for name, a, b, tol in zip(("y", "dx", "dgamma", "dbeta"), got, want, (tol_y, tol_dx, tol_g, tol_b)):
        assert a.shape == b.shape, name
        assert torch.isfinite(a).all(), name
        worst = float(((a.to(F64) - b).abs() / tol).max())
        assert worst <= 1.0, f"{name}: {worst:.3f} of the tolerance"
    return got


SHAPES = [
    ((1, 1, 1, 8), 1), ((2, 4, 4, 256), 32), ((3, 5, 7, 12), 4), ((2, 3, 3, 7), 7), ((2, 3, 3, 7), 1), ((5, 1, 1, 64), 2),
    ((2, 16, 16, 24), 3), ((2, 32, 32, 64), 8), ((1, 37, 53, 96), 8), ((3, 33, 40), 5), ((4, 48), 6), ((2, 64, 64, 32), 32),
    ((1, 100, 100, 18), 2), ((2, 96, 96, 64), 16), ((1, 40, 40, 512), 1), ((1, 20, 30, 2048), 4), ((2, 9, 1000), 8), ((1, 130, 130, 1), 1),
]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape,groups", SHAPES, ids=lambda s: str(s).replace(" ", ""))
def test_group_norm(shape, groups, dtype):
    for i, act in enumerate((None, "silu", "lrelu")):
        check(*inputs(i, shape, dtype), groups, act)


@pytest.mark.parametrize("shape,groups,dtype", [((1, 20, 30, 8192), 8192, BF16), ((2, 9, 8192), 1, BF16), ((1, 25, 20, 4096), 4096, F32),
                                                ((1, 25, 20, 4096), 2, F32), ((2, 31, 7, 1023), 1023, BF16), ((300, 3, 40), 8, F32)],
                         ids=lambda s: str(s).replace(" ", ""))
def test_the_widest_maps_and_many_samples(shape, groups, dtype):
    check(*inputs(9, shape, dtype), groups, "silu")


def test_means_far_from_zero_cost_no_digits():
    """|mean| = 1000 spreads: sums of squares would leave nothing of the variance in fp32."""
    for shape in ((2, 16, 16, 32), (1, 128, 128, 32)):
        x, gamma, beta, dy = inputs(1, shape, F32, mean=0.0)
        check(1000.0 + x, gamma, beta, dy, 4, None)


def test_constant_groups_and_eps():
    """Variance 0: n = 0, y = act(beta), dx from rstd = 1 / sqrt(eps)."""
    x, gamma, beta, dy = inputs(2, (2, 6, 6, 16), F32)
    x = torch.full_like(x, 3.0)
    y, dx, dgamma, dbeta = run(x, gamma, beta, dy, 4, None, eps=1e-2)
    assert torch.equal(y, beta.expand_as(y)) and torch.isfinite(dx).all() and float(dgamma.abs().max()) == 0.0
    check(*inputs(3, (2, 6, 6, 16), F32), 4, "silu", eps=0.5)
    check(*inputs(3, (2, 6, 6, 16), F32), 4, "lrelu", slope=0.01)


def test_group_norm_takes_other_layouts():
    x, gamma, beta, dy = inputs(4, (2, 8, 6, 32), BF16)
    base = run(x, gamma, beta, dy, 8, "silu")
    for y in (x.transpose(1, 2).contiguous().transpose(1, 2), torch.cat([x, x], -1)[..., :32]):
        got = run(y, gamma, beta, dy.transpose(1, 2).contiguous().transpose(1, 2), 8, "silu")
        assert all(torch.equal(a, b) for a, b in zip(base, got))
    # an address that is not 16-byte aligned takes the scalar form: same values, another order of summation
    buf = torch.empty(x.numel() + 8, dtype=BF16, device=DEV)
    odd = buf[1:1 + x.numel()].view(x.shape)
    odd.copy_(x)
    check(odd, gamma, beta, dy, 8, "silu")


def test_group_norm_of_nothing():
    for shape in ((0, 4, 4, 16), (2, 0, 16)):
        x, gamma, beta, dy = inputs(5, shape, BF16)
        y, dx, dgamma, dbeta = run(x, gamma, beta, dy, 4, "silu")
        assert y.shape == x.shape and dx.shape == x.shape
        assert float(dgamma.abs().max()) == 0.0 and float(dbeta.abs().max()) == 0.0


@pytest.mark.parametrize("shape", [(3, 16, 16, 64), (2, 128, 128, 64)])
def test_group_norm_repeats_replays_and_keeps_streams_apart(shape):
    sets = [inputs(10 + i, shape, BF16) for i in range(3)]
    eager = [run(*s, 8, "silu") for s in sets]
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        other = run(*sets[0], 8, "silu")
    again = run(*sets[1], 8, "silu")
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, eager[0])) and all(torch.equal(a, b) for a, b in zip(again, eager[1]))
    hold = [t.clone() for t in sets[0]]
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        run(*hold, 8, "silu")
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run(*hold, 8, "silu")
    for i in (1, 2, 0, 1):
        for t, s in zip(hold, sets[i]):
            t.copy_(s)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager[i])), i
        assert all(torch.equal(a, b) for a, b in zip(run(*sets[i], 8, "silu"), eager[i]))


def test_group_norm_gradients_against_differences():
    x, gamma, beta, dy = inputs(20, (2, 5, 6, 12), F32)
    got = run(x, gamma, beta, dy, 3, "silu")
    xs = [t.to(F64) for t in (x, gamma, beta)]
    loss = lambda a: float((ref.group_norm(*a, 3, act="silu") * dy.to(F64)).sum())
    g = torch.Generator(device=DEV).manual_seed(0)
    for i in range(3):
        d = torch.randn(xs[i].shape, generator=g, device=DEV, dtype=F64)
        up, dn = ([t + (s * 1e-5 * d if j == i else 0) for j, t in enumerate(xs)] for s in (1, -1))
        diff = (loss(up) - loss(dn)) / 2e-5
        scale = float((got[1 + i].to(F64).abs() * d.abs()).sum())
        assert abs(float((got[1 + i].to(F64) * d).sum()) - diff) <= 2.0 ** -18 * scale + 1e-6, i


def test_group_norm_refuses_second_derivatives_and_wide_scalar_maps():
    from rgbd_gan_amd import functional as Fn
    x, gamma, beta, dy = inputs(21, (1, 4, 4, 16), F32)
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(Fn.group_norm(x, gamma, beta, 4), x, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    wide = torch.zeros(1, 2, 1026, device=DEV)
    with pytest.raises(RuntimeError, match="channels"):
        Fn.group_norm(wide, torch.ones(1026, device=DEV), torch.zeros(1026, device=DEV), 2)


@pytest.mark.parametrize("shape,groups,dtype", [((2, 3, 5, 2048), 4, BF16), ((2, 3, 5, 2048), 4, F32), ((2, 40, 40, 64), 8, BF16), ((3, 7, 9, 12), 3, F32)],
                         ids=lambda s: str(s).replace(" ", ""))
def test_tensors_at_odd_addresses(shape, groups, dtype):
    """x, the output gradient or both at an address that is not 16-byte aligned: every width that is taken elsewhere is taken, and the
    numbers are the same bit for bit."""
    x, gamma, beta, dy = inputs(22, shape, dtype)
    base = check(x, gamma, beta, dy, groups, "silu")

    def odd(t):
        buf = torch.empty(t.numel() + 8, dtype=dtype, device=DEV)
        out = buf[1:1 + t.numel()].view(t.shape)
        out.copy_(t)
        assert out.is_contiguous() and out.data_ptr() % 16
        return out

    for a, d in ((x, odd(dy)), (odd(x), dy), (odd(x), odd(dy))):
        assert all(torch.equal(p, q) for p, q in zip(base, run(a, gamma, beta, d, groups, "silu")))
