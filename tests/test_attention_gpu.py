"""Grid attention (csrc/attention.hip) against its definition in 64 bits, forward and backward.

Tolerances are bounds, element by element, on what the kernels' roundings can do (U = 2^-8, half a step of bf16):
  scores      fp32 sums of D exact products and the bias: e = (D + 8) 2^-24 scale |q|.|k| + 2^-22 (|s| + cap + |bias|); a probability
              is then off by at most es = 2 max e + 2^-20 of itself (numerator and row sum)
  o           its own rounding U |o|, and the operand rounding of p: (U + es) sum p |v|   (2^-16 for U where p has two terms)
  delta       sum |do| times what o carries in fp32 plus its second term's 2^-16 |o|
  ds          operand rounding U |ds|, p's and delta's errors; through the cap (1 - tanh^2), itself off by 2^-20
  dq, dk, dv  those against |k|, |q|, |do|, and their own rounding
  dtable      ds without the operand rounding, and fp32 sums of runs of at most 64 terms: 2^-18 of the sum of magnitudes
"""
import math

import numpy as np
import pytest
import torch

from oracle import attention as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F64 = torch.bfloat16, torch.float64
U = 2.0 ** -8


def buckets(rows, cols, n=7, far=16):
    from rgbd_gan_amd.functional import RelativeBuckets
    return RelativeBuckets.log(rows, cols, n, far, device=DEV)


def inputs(seed, B, Lq, Lk, H, Hkv, D, n_buckets=0, amp=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    q, k, v = (amp * r(B, Lq, H, D)).to(BF16), r(B, Lk, Hkv, D).to(BF16), r(B, Lk, Hkv, D).to(BF16)
    return q, k, v, (r(H, n_buckets) if n_buckets else None), r(B, Lq, H, D).to(BF16)


def definition(q, k, v, table, b, do, scale, cap, lengths, q_start, fine):
    """{name: (value, tolerance)} in 64 bits."""
    m = b.map.reshape(2 * b.rows - 1, 2 * b.cols - 1).long() if b is not None else None
    q, k, v, do = (t.to(F64) for t in (q, k, v, do))
    table = table.to(F64) if table is not None else None
    B, Lq, H, D = q.shape
    Hkv, rep = k.shape[2], H // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    o, p, t, place, kr, vr = ref.attention_parts(q, k, v, table, m, scale, cap, lengths, q_start)
    qh, doh, oh = (x.permute(0, 2, 1, 3) for x in (q, do, o))
    mm = lambda a, b: torch.matmul(a, b.contiguous())
    absqk = scale * mm(qh.abs(), kr.abs().transpose(-1, -2))
    bias = table[:, place][None] if table is not None else torch.zeros(1, 1, 1, 1, dtype=F64, device=DEV)
    bias = torch.where(torch.isfinite(bias), bias, torch.zeros_like(bias))
    e = (D + 8) * 2.0 ** -24 * absqk + 2.0 ** -22 * (absqk + cap + bias.abs())
    es = 2 * float((e * (p > 0)).max()) + 2.0 ** -20 if e.numel() else 0.0
    up = 2.0 ** -16 if fine else U
    A = mm(p, vr.abs())
    back = lambda x: x.permute(0, 2, 1, 3)
    out = {"o": (o, back(U * oh.abs() + (up + es) * A) + 1e-30)}
    dp = mm(doh, vr.transpose(-1, -2))
    delta = (doh * oh).sum(-1, keepdim=True)
    edp = D * 2.0 ** -24 * mm(doh.abs(), vr.abs().transpose(-1, -2))
    edelta = (doh.abs() * ((up + es) * A + 2.0 ** -16 * oh.abs())).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    mag = p * (dp.abs() + delta.abs())
    exact_part = es * mag + p * (edp + edelta)
    E = U * ds.abs() + exact_part
    if table is not None:
        flat = place.reshape(-1)
        add = lambda x: torch.zeros(H, table.shape[1], dtype=F64, device=DEV).index_add_(1, flat, x.sum(0).reshape(H, -1))
        out["dtable"] = (add(ds), add(exact_part + 2.0 ** -18 * mag) + 1e-30)
    if cap:
        E = (1 - t * t) * E + 2.0 ** -20 * mag
        ds = ds * (1 - t * t)
    group = lambda x: back(x.reshape(B, Hkv, rep, *x.shape[2:]).sum(2))
    dq, dk, dv = scale * mm(ds, kr), scale * mm(ds.transpose(-1, -2), qh), mm(p.transpose(-1, -2), doh)
    out["dq"] = (back(dq), back(scale * mm(E, kr.abs()) + U * dq.abs()) + 1e-30)
    out["dk"] = (group(dk), group(scale * mm(E.transpose(-1, -2), qh.abs())) + U * group(dk).abs() + 1e-30)
    out["dv"] = (group(dv), group((U + es) * mm(p.transpose(-1, -2), doh.abs())) + U * group(dv).abs() + 1e-30)
    return out


def check(got, want, names):
    for n in names:
        x, (y, tol) = got[n].to(F64), want[n]
        assert x.shape == y.shape, (n, x.shape, y.shape)
        if not y.numel():
            continue
        assert torch.isfinite(x).all(), n
        worst = float(((x - y).abs() / tol).max())
        assert worst <= 1.0, f"{n}: {worst:.3f} of the tolerance"


def run(q, k, v, table, b, do, scale=None, cap=0.0, lengths=None, q_start=0):
    from rgbd_gan_amd import functional as Fn
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)] + ([table.detach().requires_grad_(True)] if table is not None else [])
    o = Fn.attention(*leaves[:3], leaves[3] if table is not None else None, b, scale, cap, lengths, q_start)
    grads = torch.autograd.grad(o, leaves, do)
    with torch.no_grad():                                       # the serving form: no second terms, no statistics kept
        plain = Fn.attention(q, k, v, table, b, scale, cap, lengths, q_start)
    return {"o": o.detach(), "plain": plain, **dict(zip(("dq", "dk", "dv", "dtable"), grads))}


def full_check(q, k, v, table, b, do, scale=None, cap=0.0, lengths=None, q_start=0):
    args = (q, k, v, table, b, do, scale, cap, lengths, q_start)
    got = run(*args)
    want = definition(*args, fine=table is not None)
    check(got, want, ["o", "dq", "dk", "dv"] + (["dtable"] if table is not None else []))
    want = definition(*args, fine=False)
    check({"o": got["plain"]}, want, ["o"])
    return got


# rows, cols, queries (0: all), q_start, keys (0: all), B, H, Hkv, D, cap, lengths
CASES = [
    (1, 1, 0, 0, 0, 2, 2, 2, 64, 0.0, None),                    # one token
    (1, 5, 0, 0, 0, 1, 1, 1, 32, 0.0, None),
    (4, 4, 0, 0, 0, 3, 4, 4, 64, 0.0, None),
    (4, 4, 0, 0, 0, 3, 4, 1, 128, 5.0, [16, 0, 1]),
    (7, 9, 0, 0, 0, 2, 3, 3, 32, 0.0, None),                    # odd columns: 4 keys straddle rows
    (7, 9, 0, 0, 0, 2, 4, 2, 64, 20.0, [63, 31]),
    (16, 16, 0, 0, 0, 2, 2, 1, 128, 0.0, [200, 256]),
    (16, 16, 0, 0, 0, 1, 2, 2, 64, 50.0, None),
    (23, 31, 0, 0, 0, 2, 2, 2, 32, 0.0, [713, 129]),
    (5, 1, 0, 0, 0, 2, 2, 2, 64, 0.0, None),                    # a single column
    (1, 129, 0, 0, 0, 2, 2, 2, 64, 0.0, [129, 65]),             # one past a block, one past a tile
    (1, 127, 0, 0, 0, 2, 6, 2, 32, 0.0, [64, 128]),             # a length beyond the keys counts them all
    (2, 1024, 0, 0, 0, 1, 1, 1, 64, 0.0, None),                 # the widest grid of more than one row
    (64, 64, 0, 0, 0, 1, 1, 1, 64, 0.0, [3000]),                # more than one window of the bias
    (33, 130, 300, 4, 0, 1, 2, 1, 32, 10.0, None),              # queries inside the grid
    (12, 12, 1, 143, 0, 2, 2, 2, 128, 0.0, [144, 7]),           # one query at the last token
    (12, 12, 0, 0, 50, 2, 2, 2, 64, 0.0, None),                 # fewer keys than queries
    (1, 3000, 5, 2995, 0, 2, 4, 2, 128, 0.0, [3000, 1024]),     # few queries over a long line
    (1, 3000, 9, 100, 0, 1, 8, 2, 64, 30.0, None),
    (9, 7, 8, 5, 40, 2, 4, 1, 32, 0.0, [40, 0]),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c).replace(" ", ""))
def test_attention_with_bias(case):
    rows, cols, lq, q0, lk, B, H, Hkv, D, cap, lens = case
    b = buckets(rows, cols, 9)
    q, k, v, table, do = inputs(1, B, lq or rows * cols, lk or rows * cols, H, Hkv, D, b.n_buckets)
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV) if lens else None
    full_check(q, k, v, table, b, do, cap=cap, lengths=lengths, q_start=q0)


@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D,cap,scale,lens", [
    (2, 1, 1, 1, 1, 32, 0.0, None, None), (1, 33, 65, 2, 1, 64, 0.0, 0.3, [40]), (2, 130, 7, 4, 4, 128, 15.0, None, [7, 3]),
    (3, 64, 192, 2, 2, 64, 0.0, None, [0, 64, 191]), (1, 200, 300, 6, 3, 32, 3.0, 1.0, None), (1, 5, 3, 1, 1, 64, 0.0, None, [0]),
    (2, 3, 2000, 4, 1, 64, 0.0, None, [2000, 77]), (1, 1, 5000, 32, 1, 128, 0.0, None, None), (1, 7, 900, 4, 1, 32, 4.0, 0.5, None)])
def test_attention_without_bias(B, Lq, Lk, H, Hkv, D, cap, scale, lens):
    q, k, v, _, do = inputs(2, B, Lq, Lk, H, Hkv, D)
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV) if lens else None
    full_check(q, k, v, None, None, do, scale=scale, cap=cap, lengths=lengths)


def test_large_scores_and_saturated_caps():
    """Scores of +-100 and a cap they saturate: the running maximum moves, tanh leaves its polynomial."""
    b = buckets(16, 16, 7)
    q, k, v, table, do = inputs(3, 2, 256, 256, 2, 2, 64, b.n_buckets, amp=12.0)
    full_check(q, k, v, table, b, do)
    full_check(q, k, v, table, b, do, cap=6.0)
    full_check(q, k, v, 30 * table, b, do, cap=40.0)


def test_rows_without_keys_are_zero_and_keys_beyond_the_length_do_not_exist():
    from rgbd_gan_amd import functional as Fn
    b = buckets(8, 10, 7)
    q, k, v, table, do = inputs(4, 3, 80, 80, 2, 1, 64, b.n_buckets)
    lengths = torch.tensor([80, 0, 37], dtype=torch.int32, device=DEV)
    k2, v2 = k.clone(), v.clone()
    for t in (k2, v2):
        t[1] = float("nan")
        t[2, 37:] = float("inf")
    a, c = (run(q, x, y, table, b, do, lengths=lengths) for x, y in ((k, v), (k2, v2)))
    for n in a:
        assert torch.equal(a[n], c[n]), n
        assert torch.isfinite(a[n]).all(), n
    for n in ("o", "plain", "dq", "dk", "dv"):
        assert float(a[n][1].float().abs().max()) == 0.0, n
    assert float(a["dk"][2, 37:].float().abs().max()) == 0.0 and float(a["dv"][2, 37:].float().abs().max()) == 0.0
    # a negative length is no length
    lengths[2] = -5
    assert float(Fn.attention(q, k, v, table, b, lengths=lengths)[2].float().abs().max()) == 0.0


def test_minus_infinity_in_the_table_masks_offsets():
    """A bias of -inf, or of the type's lowest value, takes its offsets out; a query all of whose keys it takes gives 0."""
    from rgbd_gan_amd.functional import RelativeBuckets
    rows, cols = 6, 11
    m = torch.zeros(2 * rows - 1, 2 * cols - 1, dtype=torch.long)
    m[:, cols - 1:] = 1                                           # dx >= 0
    b = RelativeBuckets(m, 2, device=DEV)
    q, k, v, _, do = inputs(5, 2, 66, 66, 2, 2, 32)
    want = definition(q, k, v, torch.tensor([[-math.inf, 0.5], [0.25, -math.inf]], device=DEV), b, do, None, 0.0, None, 0, True)
    for low in (-math.inf, torch.finfo(torch.float32).min, -1e30):
        got = run(q, k, v, torch.tensor([[low, 0.5], [0.25, low]], device=DEV), b, do)
        check(got, want, ["o", "dq", "dk", "dv", "dtable"])
        assert float(got["dtable"][0, 0]) == 0.0 and float(got["dtable"][1, 1]) == 0.0
        # head 1 sees only keys to its right: the last column has none
        assert float(got["o"].reshape(2, rows, cols, 2, 32)[:, :, -1, 1].float().abs().max()) == 0.0
    # one query row of it, over enough keys for the form that cuts them into runs
    m = torch.zeros(1, 1199, dtype=torch.long)
    m[:, 599:] = 1
    b = RelativeBuckets(m, 2, device=DEV)
    q, k, v, _, do = inputs(5, 2, 2, 600, 2, 2, 32)
    want = definition(q, k, v, torch.tensor([[-math.inf, 0.5], [0.25, -math.inf]], device=DEV), b, do, None, 0.0, None, 0, True)
    for low in (-math.inf, torch.finfo(torch.float32).min):
        check(run(q, k, v, torch.tensor([[low, 0.5], [0.25, low]], device=DEV), b, do), want, ["o", "dq", "dk", "dv", "dtable"])


def test_a_bias_far_from_zero():
    """Every score of a head moved by -3000, by +3000, by +-80: the softmax does not care, its reference has to follow."""
    b = buckets(9, 9, 7)
    q, k, v, table, do = inputs(25, 2, 81, 81, 4, 2, 64, b.n_buckets)
    shift = torch.tensor([-3000.0, 3000.0, -80.0, 80.0], device=DEV)[:, None]
    full_check(q, k, v, table + shift, b, do)
    full_check(q, k, v, table + shift, b, do, cap=9.0, lengths=torch.tensor([81, 33], dtype=torch.int32, device=DEV))


def test_scores_that_grow_and_fall_along_the_keys():
    """Scores that leave the range of the running reference in either direction, in the middle of the keys and at their end."""
    N = 400
    for sign in (1.0, -1.0):
        g = torch.Generator(device=DEV).manual_seed(26)
        r = lambda *s: torch.randn(*s, generator=g, device=DEV)
        q, k, v, do = (r(1, N, 1, 64) for _ in range(4))
        k = k + sign * torch.linspace(-12, 12, N, device=DEV)[None, :, None, None] * (torch.arange(64, device=DEV) == 3)
        q = q + 20.0 * (torch.arange(64, device=DEV) == 3)
        full_check(*(t.to(BF16) for t in (q, k, v)), None, None, do.to(BF16), scale=0.5)


def test_ties_between_bf16_neighbours():
    """o halfway between two bf16 numbers, everywhere and of either parity: its low half has to tell on which side the rounding went, or
    delta, and with it every gradient, is off by a whole step of o."""
    b = buckets(1, 2, 3)
    g = torch.Generator(device=DEV).manual_seed(27)
    v0 = torch.randn(3, 2, 64, generator=g, device=DEV).to(BF16)
    v1 = (v0.view(torch.int16) + 1).view(BF16)                          # the next one away from zero
    v = torch.stack([v0, v1], dim=1)
    q, k = torch.zeros(3, 2, 2, 64, device=DEV, dtype=BF16), torch.randn(3, 2, 2, 64, generator=g, device=DEV).to(BF16)
    do = torch.randn(3, 2, 2, 64, generator=g, device=DEV).to(BF16)
    table = torch.zeros(2, b.n_buckets, device=DEV)
    full_check(q, k, v, table, b, do)


def test_a_batch_whose_partials_are_reduced_in_pieces():
    """The table's gradient of a batch large enough for its partial sums to be reduced a few samples at a time: the other gradients
    are those of its halves bit for bit, dtable is their sum up to the order of fp32 additions."""
    for rows, cols, B, H in ((64, 64, 18, 8), (63, 65, 17, 32)):
        b = buckets(rows, cols, 7)
        q, k, v, table, do = inputs(28, B, rows * cols, rows * cols, H, H, 32, b.n_buckets)
        lengths = torch.randint(1, rows * cols, (B,), dtype=torch.int32, device=DEV)
        whole = run(q, k, v, table, b, do, lengths=lengths)
        h = B // 2
        parts = [run(*(t[s] for t in (q, k, v)), table, b, do[s], lengths=lengths[s]) for s in (slice(0, h), slice(h, B))]
        for n in ("o", "dq", "dk", "dv"):
            assert torch.equal(whole[n], torch.cat([x[n] for x in parts])), (rows, n)
        both = parts[0]["dtable"].double() + parts[1]["dtable"].double()
        assert float((whole["dtable"].double() - both).norm() / both.norm()) <= 2.0 ** -18


def test_strides_orders_and_packed_layouts():
    """q, k, v as views of one projection, with heads before tokens, with a shared batch, and at an offset that is not 16-byte
    aligned: the same numbers as contiguous tensors; the packed form's gradient has the packed layout."""
    from rgbd_gan_amd import functional as Fn
    b = buckets(5, 12, 7)
    B, N, H, Hkv, D = 2, 60, 4, 2, 64
    q, k, v, table, do = inputs(6, B, N, N, H, Hkv, D, b.n_buckets)
    base = run(q, k, v, table, b, do)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    odd = []
    for t in (q, k, v):
        buf = torch.empty(t.numel() + 8, dtype=BF16, device=DEV)
        odd.append(buf[3:3 + t.numel()].view(t.shape))
        odd[-1].copy_(t)
    for alt in (heads_first, odd):
        got = run(*alt, table, b, do.transpose(1, 2).contiguous().transpose(1, 2))
        for n in base:
            assert torch.equal(base[n], got[n]), n
    for shape in ((B, N, -1), (B, 5, 12, -1)):
        qkv = torch.cat([t.flatten(2) for t in (q, k, v)], dim=-1).reshape(shape).requires_grad_(True)
        leaf = table.detach().requires_grad_(True)
        o = Fn.attention_packed(qkv, H, Hkv, leaf, b)
        dqkv, dt = torch.autograd.grad(o, (qkv, leaf), do)
        assert torch.equal(o, base["o"]) and torch.equal(dt, base["dtable"]) and dqkv.shape == qkv.shape
        want = torch.cat([base[n].flatten(2) for n in ("dq", "dk", "dv")], dim=-1).reshape(shape)
        assert torch.equal(dqkv, want)
        assert torch.equal(Fn.attention_packed(qkv.detach(), H, Hkv, table, b), base["plain"])
    # an output gradient at an odd address, and one that is a single number for all
    buf = torch.empty(do.numel() + 8, dtype=BF16, device=DEV)
    odd_do = buf[5:5 + do.numel()].view(do.shape)
    odd_do.copy_(do)
    got = run(q, k, v, table, b, odd_do)
    assert all(torch.equal(base[n], got[n]) for n in base)
    got, ones = run(q, k, v, table, b, torch.ones(1, 1, 1, 1, dtype=BF16, device=DEV).expand(do.shape)), run(q, k, v, table, b, torch.ones_like(do))
    assert all(torch.equal(ones[n], got[n]) for n in ones)
    # one k, v for the whole batch (stride 0) and its summed gradient
    k1, v1 = (t[:1].clone().requires_grad_(True) for t in (k, v))
    # (a table that is learned: its gradient asks for the finer second product, as in run())
    o = Fn.attention(q, k1.expand(B, -1, -1, -1), v1.expand(B, -1, -1, -1), table.detach().requires_grad_(True), b)
    dk, dv = torch.autograd.grad(o, (k1, v1), do)
    whole = run(q, k[:1].expand(B, -1, -1, -1).contiguous(), v[:1].expand(B, -1, -1, -1).contiguous(), table, b, do)
    assert torch.equal(o, whole["o"])
    for x, n in ((dk, "dk"), (dv, "dv")):
        s = whole[n].to(F64).sum(0, keepdim=True)
        # torch sums the expanded gradient in fp32 and rounds to bf16 once
        assert float(((x.to(F64) - s).abs() / (U * s.abs() + 2.0 ** -22 * whole[n].to(F64).abs().sum(0, keepdim=True) + 1e-30)).max()) <= 1.0


def test_empty_shapes():
    from rgbd_gan_amd import functional as Fn
    b = buckets(3, 4, 7)
    for B, Lq, Lk in ((0, 5, 5), (2, 0, 5), (2, 5, 0), (2, 0, 0)):
        q, k, v, table, do = inputs(7, B, Lq, Lk, 2, 2, 64, b.n_buckets)
        got = run(q, k, v, table, b, do)
        assert got["o"].shape == q.shape and got["dk"].shape == k.shape
        for n in got:
            assert float(got[n].float().abs().sum()) == 0.0, (B, Lq, Lk, n)
    q, k, v, _, do = inputs(7, 2, 3, 0, 2, 2, 64)
    assert float(run(q, k, v, None, None, do)["o"].float().abs().sum()) == 0.0
    # a grid without columns cannot be built; lengths of an empty batch are fine
    q, k, v, table, do = inputs(7, 0, 4, 4, 2, 2, 64, b.n_buckets)
    assert Fn.attention(q, k, v, table, b, lengths=torch.empty(0, dtype=torch.int32, device=DEV)).shape == (0, 4, 2, 64)


def test_results_repeat_bit_for_bit_and_streams_keep_their_own():
    b = buckets(20, 20, 9)
    q, k, v, table, do = inputs(8, 3, 400, 400, 4, 2, 64, b.n_buckets)
    base = run(q, k, v, table, b, do, cap=20.0)
    q2, k2, v2, t2, do2 = inputs(9, 3, 400, 400, 4, 2, 64, b.n_buckets)
    base2 = run(q2, k2, v2, t2, b, do2, cap=20.0)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s1):
            a = run(q, k, v, table, b, do, cap=20.0)
        with torch.cuda.stream(s2):
            c = run(q2, k2, v2, t2, b, do2, cap=20.0)
        torch.cuda.synchronize()
        for n in base:
            assert torch.equal(a[n], base[n]) and torch.equal(c[n], base2[n]), n


def test_captured_graphs_replay_with_new_inputs():
    """Two graphs of the training pass, replayed in turn with new inputs and the eager pass in between."""
    from rgbd_gan_amd import functional as Fn
    b = buckets(9, 14, 7)
    sets = [inputs(10 + i, 2, 126, 126, 2, 1, 64, b.n_buckets) for i in range(4)]
    lens = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([126, 60], [0, 126], [126, 126], [1, 5])]

    def passes(q, k, v, table, do, lengths):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
        o = Fn.attention(*leaves, b, lengths=lengths)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    eager = [passes(*s, l) for s, l in zip(sets, lens)]
    graphs = []
    for i in range(2):
        hold = [t.clone() for t in sets[i]] + [lens[i].clone()]
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            passes(*hold)
        torch.cuda.current_stream().wait_stream(st)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = passes(*hold)
        graphs.append((g, hold, out))
    for rep in range(4):
        for i, (g, hold, out) in enumerate(graphs):
            j = (rep + 2 * i) % 4
            for t, s in zip(hold, list(sets[j]) + [lens[j]]):
                t.copy_(s)
            g.replay()
            torch.cuda.synchronize()
            for x, y in zip(out, eager[j]):
                assert torch.equal(x, y), (rep, i)
            again = passes(*sets[j], lens[j])
            assert all(torch.equal(x, y) for x, y in zip(again, eager[j]))


def test_other_forms_captured_and_replayed():
    """The forms that the sizes above do not reach: keys in runs (few queries), queries in runs (few keys), offsets by diagonals and by
    blocks, a table without gradient; each captured, replayed with new inputs, the eager pass in between."""
    from rgbd_gan_amd import functional as Fn
    for rows, cols, lq, H, Hkv, D, learned in ((1, 1400, 3, 4, 1, 64, True), (33, 20, 0, 8, 2, 32, True), (32, 32, 0, 1, 1, 128, True),
                                              (16, 20, 0, 2, 2, 64, False)):
        n = rows * cols
        lq = lq or n
        b = buckets(rows, cols, 7)
        sets = [inputs(40 + i, 2, lq, n, H, Hkv, D, b.n_buckets) for i in range(3)]
        lens = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([n, 60], [0, n], [n - 1, 1])]

        def passes(q, k, v, table, do, lengths):
            leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
            table = table.detach().requires_grad_(learned)
            o = Fn.attention(*leaves, table, b, lengths=lengths, q_start=n - lq)
            return (o.detach(), *torch.autograd.grad(o, leaves + [table] * learned, do))

        eager = [passes(*s, l) for s, l in zip(sets, lens)]
        hold = [t.clone() for t in sets[0]] + [lens[0].clone()]
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            passes(*hold)
        torch.cuda.current_stream().wait_stream(st)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = passes(*hold)
        for j in (1, 2, 0, 1):
            for t, s in zip(hold, list(sets[j]) + [lens[j]]):
                t.copy_(s)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, eager[j])), (rows, cols, j)
            assert all(torch.equal(x, y) for x, y in zip(passes(*sets[j], lens[j]), eager[j]))


def test_nothing_is_read_that_was_not_written():
    """Memory that held NaN before a call (workspaces, statistics, outputs) changes nothing."""
    for rows, cols, lq, lk, B, H, Hkv, D, lens in (
            (1, 1400, 3, 0, 2, 4, 1, 64, [1400, 9]), (33, 20, 0, 0, 2, 8, 2, 32, [0, 321]), (32, 32, 0, 0, 2, 2, 1, 128, [1024, 70]),
            (64, 64, 130, 0, 1, 1, 1, 64, [2000]), (1, 300, 0, 0, 3, 2, 2, 64, [300, 1, 0]), (12, 20, 50, 100, 2, 2, 2, 64, [40, 100]),
            (32, 32, 64, 900, 1, 2, 2, 64, None), (7, 8, 0, 0, 2, 2, 1, 32, [56, 3])):
        n = rows * cols
        lq, lk = lq or n, lk or n
        b = buckets(rows, cols, 7)
        q, k, v, table, do = inputs(50, B, lq, lk, H, Hkv, D, b.n_buckets)
        lengths = torch.tensor(lens, dtype=torch.int32, device=DEV) if lens is not None else None
        args = dict(lengths=lengths, q_start=n - lq)
        want = definition(q, k, v, table, b, do, None, 0.0, lengths, n - lq, True)
        for size in (1 << 8, 1 << 14, 1 << 18, 1 << 21, 1 << 23):        # blocks of every pool the allocator gives out again
            held = [torch.full((size,), math.nan, device=DEV) for _ in range(8)]
            del held
        check(run(q, k, v, table, b, do, **args), want, ["o", "dq", "dk", "dv", "dtable"])


def test_many_samples_of_few_queries_and_runs_of_queries():
    """Enough samples for one run of keys each (the rows are written by the first launch), and shapes on either side of cutting the
    queries of dk and dv into runs."""
    b = buckets(20, 21, 7)
    for B, lq, H, Hkv, D, lens in ((300, 1, 4, 2, 64, None), (260, 3, 8, 1, 32, True), (300, 2, 2, 1, 128, True)):
        q, k, v, table, do = inputs(70, B, lq, 420, H, Hkv, D, b.n_buckets)
        lengths = torch.arange(B, dtype=torch.int32, device=DEV) * 3 % 421 if lens else None
        full_check(q, k, v, table, b, do, lengths=lengths, q_start=11)
    for B, n, H, Hkv, D in ((2, 700, 6, 2, 32), (1, 520, 16, 1, 64), (1, 513, 4, 1, 128), (1, 500, 4, 4, 64)):
        q, k, v, _, do = inputs(71, B, n, n, H, Hkv, D)
        full_check(q, k, v, None, None, do, lengths=torch.tensor([n - 7] * B, dtype=torch.int32, device=DEV))


def test_keys_in_runs():
    """Few workgroups: runs of two tiles and more, lengths that leave runs empty or short, every way the table's sums are taken."""
    for rows, cols, lq, H, Hkv, D, cap, lens in ((20, 20, 0, 2, 1, 64, 0.0, [400, 130, 0]), (32, 32, 0, 2, 2, 64, 9.0, [1024, 1]),
                                                (1, 1000, 300, 4, 2, 128, 0.0, [999, 64]), (19, 33, 200, 2, 2, 32, 4.0, [627, 65]),
                                                (64, 64, 100, 1, 1, 32, 0.0, [4096]), (8, 40, 0, 2, 2, 128, 0.0, None)):
        n = rows * cols
        lq = lq or n
        B = len(lens) if lens else 2
        b = buckets(rows, cols, 9)
        q, k, v, table, do = inputs(80, B, lq, n, H, Hkv, D, b.n_buckets)
        lengths = torch.tensor(lens, dtype=torch.int32, device=DEV) if lens else None
        full_check(q, k, v, table, b, do, cap=cap, lengths=lengths, q_start=(n - lq) // 2)
    # scores far apart between the runs, rows of which one run has no key or all
    b = buckets(1, 1000, 9, 500)
    q, k, v, table, do = inputs(82, 1, 1000, 1000, 1, 1, 64, b.n_buckets)
    for far in (300.0, -300.0, -math.inf):
        t = table.clone()
        t[0, 0] += far
        t[0, 8] -= far if far > -math.inf else -7.0
        got = run(q, k, v, t, b, do)
        check(got, definition(q, k, v, t, b, do, None, 0.0, None, 0, True), ["o", "dq", "dk", "dv", "dtable"])
    q, k, v, _, do = inputs(81, 1, 300, 2000, 2, 2, 64)
    full_check(q, k, v, None, None, do, lengths=torch.tensor([1234], dtype=torch.int32, device=DEV))


def test_a_negative_scale_is_a_negative_query():
    b = buckets(9, 13, 7)
    q, k, v, table, do = inputs(60, 2, 117, 117, 4, 2, 64, b.n_buckets)
    for cap in (0.0, 6.0):
        got = run(q, k, v, table, b, do, scale=-0.3, cap=cap)
        got["dq"] = -got["dq"]
        check(got, definition(-q, k, v, table, b, do, 0.3, cap, None, 0, True), ["o", "dq", "dk", "dv", "dtable"])


def test_a_table_without_gradient():
    from rgbd_gan_amd import functional as Fn
    b = buckets(13, 11, 7)
    q, k, v, table, do = inputs(61, 2, 143, 143, 2, 1, 64, b.n_buckets)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = Fn.attention(*leaves, table, b, cap=12.0)
    got = {"o": o.detach(), **dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)))}
    check(got, definition(q, k, v, table, b, do, None, 12.0, None, 0, False), list(got))


def test_gradients_against_differences():
    """<gradient, direction> against central differences of the 64-bit definition, h small enough for their own error to vanish
    next to the tolerance summed over the direction."""
    b = buckets(6, 7, 7)
    q, k, v, table, do = inputs(20, 2, 42, 42, 4, 2, 32, b.n_buckets)
    lengths = torch.tensor([42, 20], dtype=torch.int32, device=DEV)
    got = run(q, k, v, table, b, do, cap=8.0, lengths=lengths)
    want = definition(q, k, v, table, b, do, None, 8.0, lengths, 0, True)
    m = b.map.reshape(11, 13).long()
    x = [t.to(F64) for t in (q, k, v, table)]
    loss = lambda xs: float((ref.attention(*xs, m, cap=8.0, lengths=lengths) * do.to(F64)).sum())
    g = torch.Generator(device=DEV).manual_seed(0)
    for i, n in enumerate(("dq", "dk", "dv", "dtable")):
        d = torch.randn(x[i].shape, generator=g, device=DEV, dtype=F64)
        h = 1e-5
        up, dn = ([t + (s * h * d if j == i else 0) for j, t in enumerate(x)] for s in (1, -1))
        diff = (loss(up) - loss(dn)) / (2 * h)
        tol = float((want[n][1] * d.abs()).sum()) + 1e-6 * abs(diff) + 1e-6
        assert abs(float((got[n].to(F64) * d).sum()) - diff) <= tol, n


def test_second_derivatives_and_other_devices_are_refused():
    from rgbd_gan_amd import functional as Fn
    q, k, v, _, do = inputs(21, 1, 8, 8, 1, 1, 32)
    q.requires_grad_(True)
    (dq,) = torch.autograd.grad(Fn.attention(q, k, v), q, do, create_graph=True)
    with pytest.raises(RuntimeError):
        dq.float().sum().backward()
    with pytest.raises(RuntimeError, match="int32"):
        Fn.attention(q, k, v, lengths=torch.ones(1, dtype=torch.int64, device=DEV))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        Fn.attention(q, k, v, lengths=torch.ones(1, dtype=torch.int32))


def test_offsets_beyond_two_to_the_31():
    """The last sample of a batch whose tensors pass 2^31 elements (batch stride far apart, little memory touched)."""
    from rgbd_gan_amd import functional as Fn
    N, H, D = 20, 2, 64
    big = torch.empty((1 << 31) + (1 << 20), dtype=BF16, device=DEV)
    q, k, v, _, do = inputs(22, 2, N, N, H, H, D)
    views = []
    for i, t in enumerate((q, k, v)):
        w = big.as_strided((2, N, H, D), ((1 << 31) + 8 * 1024, H * D, D, 1), i * 16384)
        w.copy_(t)
        views.append(w)
    assert torch.equal(Fn.attention(*views), Fn.attention(q, k, v))
    a, c = run(*views, None, None, do), run(q, k, v, None, None, do)
    for n in a:
        assert torch.equal(a[n], c[n]), n


@pytest.mark.parametrize("far,size", [(35.0, 1e22), (-50.0, 1e-18), (0.0, 1e29), (0.0, 1e-27), (16.0, 1e29), (-6.0, 1e-27), (-25.0, 1e-27),
                                      (-31.0, 1e-27)])
def test_values_far_from_one(far, size):
    """Scores and values both away from 1: the output is finite and keeps its digits, whatever the sum of the exponentials times a value
    would be.  The whole form, keys in runs, few queries."""
    for rows, cols, lq, H, Hkv, D in ((9, 9, 81, 2, 1, 64), (1, 1000, 300, 2, 1, 128), (1, 3000, 5, 2, 1, 32)):
        n = rows * cols
        b = buckets(rows, cols, 9)
        q, k, v, table, do = inputs(90, 2, lq, n, H, Hkv, D, b.n_buckets)
        lengths = torch.tensor([n, n - 13], dtype=torch.int32, device=DEV)
        full_check(q, k, (size * v.float()).to(BF16), table + far, b, do, lengths=lengths, q_start=n - lq)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("keys", [1, 2, 5])
def test_the_learned_tables_forward_pass_keeps_fp32_digits(keys, D):
    """With a learned table o and its low half are one fp32 number, and the probabilities enter its product in three bf16 terms.  Queries
    of zero leave the bias, within +-1, as the score.  A term leaves U of what it rounds, so three leave 2^-24 of a probability; the
    product adds at most 15 terms (2^-24 each), then the division, its product and the low half: within 2^-19 of sum p |v|, and es, the
    scores' share (2 x 2^-22 |bias| + 2^-20).  Two terms would leave up to 2^-16.  One key: o is v, and its table's gradient, do . v - do . o,
    is 0; do has one channel, so that dp is exact and delta o's error."""
    from rgbd_gan_amd import functional as Fn
    from rgbd_gan_amd import kernels
    N, H = 200, 4
    b = Fn.RelativeBuckets(np.arange(2 * N - 1)[None, :], device=DEV)
    g = torch.Generator(device=DEV).manual_seed(91)
    q = torch.zeros(2, N, H, D, device=DEV, dtype=BF16)
    k, v = (torch.randn(2, keys, H, D, generator=g, device=DEV).to(BF16) for _ in range(2))
    table = 2 * torch.rand(H, b.n_buckets, generator=g, device=DEV) - 1
    o, lo, _ = kernels.attention_fwd(kernels.AttnOperands.of(q, k, v), table, b, keep=True, fine=True)
    whole = ((o.view(torch.int16).to(torch.int32) << 16) + lo.view(torch.int16).to(torch.int32)).view(torch.float32).to(F64)
    want, p, _, _, _, vr = ref.attention_parts(q.to(F64), k.to(F64), v.to(F64), table.to(F64), b.map.reshape(1, -1).long())
    tol = (2 * 2.0 ** -22 + 2.0 ** -20 + 2.0 ** -19) * torch.matmul(p, vr.abs()).permute(0, 2, 1, 3)
    worst = float(((whole - want).abs() / tol).max())
    assert worst <= 1.0, f"{worst:.3f} of the tolerance"
    if keys == 1:
        do = torch.zeros_like(q)
        do[0, :, :, 3] = torch.randn(N, H, generator=g, device=DEV).to(BF16)
        got = run(q, k, v, table, b, do)["dtable"]
        first = N - 1                                            # query i, key 0: offset i
        bound = (2 * 2.0 ** -22 + 2.0 ** -20 + 2.0 ** -19 + 2.0 ** -23) * (do[0, :, :, 3].to(F64).abs() * v[0, :, :, 3].to(F64).abs()).T
        assert float((got[:, first:].to(F64).abs() / bound.clamp_min(1e-30)).max()) <= 1.0
        assert float(got[:, :first].abs().max()) == 0.0


@pytest.mark.parametrize("rows,cols,lq,B,H,Hkv,D,cap", [(32, 32, 0, 3, 4, 4, 64, 0.0), (64, 64, 0, 1, 2, 2, 64, 30.0), (23, 31, 0, 3, 6, 2, 32, 20.0),
                                                        (1, 1500, 0, 2, 4, 2, 128, 0.0), (1, 3000, 5, 2, 4, 2, 64, 0.0), (16, 16, 0, 4, 4, 4, 64, 50.0)])
def test_the_tables_gradient_against_64_bits(rows, cols, lq, B, H, Hkv, D, cap):
    """dtable in relative 2-norm, by blocks, by diagonals, for few queries.  A pair's ds is off by independent roundings of 2^-24: the
    square root of D of them in each product, some 8 more on the way (bias, cap, exponential, delta), of magnitudes |dp| + |delta| up to
    twice ds: (sqrt(128) + 8) 2^-24 x 2 < 2^-18.5 of it, and sums of independent errors keep that ratio.  One bf16 term instead of three
    gives 5e-4."""
    n = rows * cols
    b = buckets(rows, cols, 15, 64)
    q, k, v, table, do = inputs(92, B, lq or n, n, H, Hkv, D, b.n_buckets)
    got = run(q, k, v, table, b, do, cap=cap, q_start=n - (lq or n))["dtable"].to(F64)
    m = b.map.reshape(2 * rows - 1, 2 * cols - 1).long()
    leaf = table.to(F64).requires_grad_(True)
    o = ref.attention(*(t.to(F64) for t in (q, k, v)), leaf, m, cap=cap, q_start=n - (lq or n))
    (want,) = torch.autograd.grad(o, leaf, do.to(F64))
    err = float((got - want).norm() / want.norm())
    print(f"dtable {rows}x{cols} lq={lq} D={D} cap={cap}: {err:.2e}", flush=True)
    assert err <= 2.0 ** -18.5
