"""CPU side of group norm and grid attention: refusals, the bucket plan, the 64-bit oracle against differences."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import attention as ref

BF16, F64 = torch.bfloat16, torch.float64


def bf(*shape):
    return torch.zeros(*shape, dtype=BF16)


def log_map(rows, cols, n=7):
    from rgbd_gan_amd.functional import RelativeBuckets
    return RelativeBuckets.log(rows, cols, n, 16, device="cpu")


# ------------------------------------------------------------------------------------------------ bucket plan
def test_buckets_list_every_offset_once():
    from rgbd_gan_amd.functional import RelativeBuckets
    rng = np.random.RandomState(0)
    m = rng.randint(0, 5, (7, 11))
    m[m == 3] = 4                                              # an empty bucket
    b = RelativeBuckets(m, 6, device="cpu")
    assert (b.rows, b.cols, b.n_buckets) == (4, 6, 6)
    assert b.map.dtype == b.order.dtype == b.start.dtype == torch.int32
    assert b.start.tolist()[0] == 0 and b.start.tolist()[-1] == m.size and b.start.numel() == 7
    for u in range(6):
        got = b.order[b.start[u]:b.start[u + 1]].tolist()
        assert got == np.nonzero(m.reshape(-1) == u)[0].tolist()


@pytest.mark.parametrize("rows,cols,n", [(1, 1, 3), (1, 200, 9), (5, 1, 5), (8, 8, 15), (9, 33, 7)])
def test_log_buckets_keep_the_sign_and_grow(rows, cols, n):
    from rgbd_gan_amd.functional import RelativeBuckets
    b = RelativeBuckets.log(rows, cols, n, 16, device="cpu")
    m = b.map.reshape(2 * rows - 1, 2 * cols - 1).numpy()
    x = m[rows - 1] - (m[rows - 1, cols - 1] // n * n if rows > 1 else 0)       # dy = 0
    assert b.n_buckets == (n if rows == 1 else n * n)
    assert (np.diff(x) >= 0).all() and x[cols - 1] == n // 2
    assert (x + x[::-1] == n - 1).all()                                        # bucket(-d) mirrors bucket(d)


@pytest.mark.parametrize("bad", [np.zeros((2, 3), int), np.zeros((3, 4), int), np.zeros((3,), int), np.zeros((3, 3)),
                                 np.full((3, 3), -1), np.full((3, 3), 9)])
def test_bad_bucket_maps_are_refused(bad):
    from rgbd_gan_amd.functional import RelativeBuckets
    with pytest.raises(ValueError):
        RelativeBuckets(bad, 9, device="cpu")


def test_log_buckets_refuse_even_counts():
    from rgbd_gan_amd.functional import RelativeBuckets
    for n in (1, 2, 8):
        with pytest.raises(ValueError):
            RelativeBuckets.log(4, 4, n, device="cpu")


# ------------------------------------------------------------------------------------------------ refusals
def test_attention_refuses_what_it_cannot_compute():
    from rgbd_gan_amd import functional as Fn
    q, k = bf(2, 6, 4, 64), bf(2, 9, 2, 64)
    b = log_map(3, 3)
    table = torch.zeros(4, b.n_buckets)
    cases = [
        (dict(q=q.float()), "bf16"),
        (dict(q=bf(2, 6, 4, 48), k=bf(2, 9, 2, 48), v=bf(2, 9, 2, 48)), "head size"),
        (dict(q=bf(2, 6, 4 * 64)), r"\(B, tokens"),
        (dict(v=bf(2, 8, 2, 64)), "do not match"),
        (dict(q=bf(3, 6, 4, 64)), "do not match"),
        (dict(k=bf(2, 9, 3, 64), v=bf(2, 9, 3, 64)), "do not divide"),
        (dict(cap=-1.0), "cap"),
        (dict(cap=float("nan")), "cap"),
        (dict(cap=float("inf")), "cap"),
        (dict(cap=1e-35), "cap"),
        (dict(cap=1e13), "cap"),
        (dict(scale=0.0), "scale"),
        (dict(scale=float("nan")), "scale"),
        (dict(scale=float("inf")), "scale"),
        (dict(table=table), "come together"),
        (dict(buckets=b), "come together"),
        (dict(table=table[:3], buckets=b), "table must be"),
        (dict(table=table, buckets=b, q_start=4), "outside"),
        (dict(table=table, buckets=b, q_start=-1), "outside"),
        (dict(table=table, buckets=log_map(2, 2)), "outside"),
        (dict(table=torch.zeros(4, 49), buckets=log_map(2, 1500)), "1024 columns"),
        (dict(q_start=1), "needs a table"),
        (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
        (dict(), "GPU tensor"),
    ]
    for change, word in cases:
        kw = dict(q=q, k=k, v=k, **{n: t for n, t in change.items() if n not in "qkv"})
        kw.update({n: t for n, t in change.items() if n in "qkv"})
        with pytest.raises(RuntimeError, match=word):
            Fn.attention(**kw)


def test_attention_packed_refuses_widths_that_do_not_split():
    from rgbd_gan_amd import functional as Fn
    for x, h, kv in ((bf(2, 6, 100), 4, 4), (bf(2, 6), 1, 1), (bf(2, 6, 384), 0, 1), (bf(2, 6, 384), 2, 0)):
        with pytest.raises(RuntimeError, match="split"):
            Fn.attention_packed(x, h, kv)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        Fn.attention_packed(bf(2, 3, 3, 3 * 128), 2)


def test_group_norm_refuses_what_it_cannot_compute():
    from rgbd_gan_amd import functional as Fn
    x, g = bf(2, 4, 4, 12), torch.ones(12)
    for args, word in (((x, g, g, 5), "divide"), ((x, g, g, 0), "divide"), ((x, g[:6], g, 3), "gamma"), ((x, g, g[:1], 3), "beta"),
                       ((x.half(), g, g, 3), "bf16 or fp32"), ((x, g, g, 3), "GPU tensor"), ((g, g, g, 3), "batch")):
        with pytest.raises(RuntimeError, match=word):
            Fn.group_norm(*args)
    with pytest.raises(RuntimeError, match="act"):
        Fn.group_norm(x, g, g, 3, act="gelu")


def test_c_entries_report_bad_arguments():
    from rgbd_gan_amd import _lib, kernels
    lib = _lib.load()
    assert lib.rgbd_group_norm_workspace(2, 16, 12, 5, 0, 0) == -1 and b"divide" in lib.rgbd_last_error()
    assert lib.rgbd_group_norm_workspace(2, 16, 12, 3, 2, 0) == -1 and b"dtype" in lib.rgbd_last_error()
    assert lib.rgbd_group_norm_workspace(2, 16, 12, 3, 0, 1) > 0
    assert lib.rgbd_group_norm_fwd(None, None, None, None, None, None, None, 2, 16, 12, 3, 0, 0, 1e-5, 0.2, None) == -1
    assert b"null" in lib.rgbd_last_error()
    assert lib.rgbd_group_norm_fwd(None, None, None, None, None, None, None, 2, 16, 12, 3, 0, 3, 1e-5, 0.2, None) == -1
    assert lib.rgbd_group_norm_fwd(None, None, None, None, None, None, None, 0, 16, 12, 3, 0, 0, 1e-5, 0.2, None) == 0
    # a width that only fits 16-byte vectors, at an address that is not 16-byte aligned
    assert lib.rgbd_group_norm_fwd(8, 16, 16, 16, 16, 16, 16, 2, 16, 2048, 4, 0, 0, 1e-5, 0.2, None) == -1
    assert b"channels" in lib.rgbd_last_error()
    assert lib.rgbd_group_norm_bwd(16, 8, 16, 16, 16, 16, 16, 16, 16, 16, 2, 16, 2048, 4, 0, 0, 0.2, None) == -1
    assert lib.rgbd_attention_fwd(None, None, None, None, None) == -1
    d = kernels._AttnDesc()
    d.B, d.H, d.Hkv, d.Lq, d.Lk, d.D, d.scale = 1, 2, 1, 4, 4, 64, 0.125
    ok = lambda: lib.rgbd_attention_bwd_workspace(ctypes.byref(d), 0)
    assert ok() > 0
    for name, value in (("D", 40), ("Hkv", 3), ("H", 0), ("Lq", -1), ("cap", -1.0), ("cap", float("nan")), ("scale", 0.0), ("q_sl", 4), ("k_sl", 1 << 24),
                        ("v_sl", -64), ("k", 8), ("B", 1 << 22), ("scale", 1e13)):
        old = getattr(d, name)
        setattr(d, name, value)
        assert ok() == -1, name
        setattr(d, name, old if old is not None else None)
    assert ok() > 0
    d.table = 16                                                # a table without its map, then a bad grid
    assert ok() == -1
    d.map, d.n_buckets, d.rows, d.cols = 16, 4, 1, 3
    assert ok() == -1 and b"outside" in lib.rgbd_last_error()
    d.cols = 4
    assert ok() > 0
    assert lib.rgbd_attention_fwd(ctypes.byref(d), None, None, None, None) == -1 and b"null" in lib.rgbd_last_error()
    assert lib.rgbd_attention_bwd(ctypes.byref(d), None, None, None) == -1
    g = kernels._AttnGrad()
    assert lib.rgbd_attention_bwd(ctypes.byref(d), ctypes.byref(g), None, None) == -1 and b"null" in lib.rgbd_last_error()


def test_the_descriptors_match_the_header_in_size():
    """3 pointers, 9 strides, 4 pointers, 10 ints, 2 floats, 1 int (padded to 8) and 6 pointers, 9 strides, 3 pointers."""
    from rgbd_gan_amd import kernels
    assert ctypes.sizeof(kernels._AttnDesc) == 8 * (3 + 9 + 4) + 4 * (10 + 2 + 1) + 4
    assert ctypes.sizeof(kernels._AttnGrad) == 8 * (6 + 9 + 3)


# ------------------------------------------------------------------------------------------------ the oracle itself
def test_oracle_attention_gradients_match_differences():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=F64).requires_grad_(True)
    b = log_map(3, 4, 5)
    m = b.map.reshape(5, 7).long()
    q, k, v, table = r(2, 5, 4, 3), r(2, 12, 2, 3), r(2, 12, 2, 3), r(4, 25)
    lengths = torch.tensor([12, 0])
    fn = lambda q, k, v, table: ref.attention(q, k, v, table, m, cap=2.0, lengths=lengths, q_start=6)
    assert torch.autograd.gradcheck(fn, (q, k, v, table), eps=1e-6, atol=1e-7)
    assert float(fn(q, k, v, table)[1].abs().max()) == 0.0


@pytest.mark.parametrize("act", [None, "silu", "lrelu"])
def test_oracle_group_norm_gradients_match_differences(act):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=F64).requires_grad_(True)
    assert torch.autograd.gradcheck(lambda x, a, b: ref.group_norm(x, a, b, 2, act=act), (r(2, 3, 2, 6), r(6), r(6)), eps=1e-6, atol=1e-6)


# ------------------------------------------------------------------------------------------------ the generator's option
def test_self_attention_option():
    from rgbd_gan_amd.net import attention_sizes
    from rgbd_gan_amd.training import setup_generator
    from rgbd_gan_amd.utils.yaml_utils import Config
    for value, want in ((None, []), (0, []), (32, [32]), ([32, 16], [16, 32]), ("16, 32", [16, 32]), ("64", [64]), ("", [])):
        assert attention_sizes(value, 6) == want
    for bad in (24, 256, [16, 5], "2"):
        with pytest.raises(ValueError):
            attention_sizes(bad, 6)
    for arch in ("dcgan", "deepvoxels"):
        with pytest.raises(AssertionError, match="self_attention"):
            setup_generator(Config(dict(generator_architecture=arch, ch=256, self_attention=32)), "cpu")


def test_partial_sums_of_the_table_stay_below_their_limit():
    """The table gradient's partial sums take 512 MB, or what one sample takes where that is more: workspace floats of a batch against
    those of one sample, whatever the batch (the rest of the difference is delta and runs of keys or queries, which want_table = 0 has too)."""
    from rgbd_gan_amd import _lib, kernels
    lib = _lib.load()
    for rows, cols, H, D in ((128, 128, 6, 64), (64, 64, 8, 32), (100, 100, 3, 64), (63, 65, 32, 32), (1, 20000, 2, 128)):
        d = kernels._AttnDesc()
        d.H, d.Hkv, d.Lq, d.Lk, d.D, d.scale, d.table, d.map = H, H, rows * cols, rows * cols, D, 0.125, 16, 16
        d.rows, d.cols, d.n_buckets = rows, cols, 9

        def floats(B):
            d.B = B
            return lib.rgbd_attention_bwd_workspace(ctypes.byref(d), 1) - lib.rgbd_attention_bwd_workspace(ctypes.byref(d), 0)

        one = floats(1)                                          # partials and what the first reduction leaves: at most 16 a head and token
        for B in (2, 3, 5, 18, 40):
            assert 0 < floats(B) <= max((128 << 20) + 16 * H * rows * cols, one), (rows, cols, H, B, floats(B), one)


# ------------------------------------------------------------------------------------------------ derivatives that are not there
def test_forward_mode_derivatives_are_refused(monkeypatch):
    """A tangent on any input raises, whether or not gradients are recorded; without one a dual level changes nothing.  (The kernels'
    wrappers are replaced: the refusal needs no GPU.)"""
    import torch.autograd.forward_ad as ad
    from rgbd_gan_amd import functional as Fn
    from rgbd_gan_amd import kernels
    monkeypatch.setattr(kernels, "group_norm_fwd", lambda x, *a: (torch.empty_like(x), torch.empty(4)))
    monkeypatch.setattr(kernels, "attention_fwd", lambda op, *a, **kw: (torch.empty_like(op.tensors[0]),) * 3)
    x, g, q = bf(2, 3, 16), torch.ones(16), bf(2, 4, 2, 64)
    b = log_map(2, 2)
    table = torch.zeros(2, b.n_buckets)
    calls = {
        "x": (x, lambda t: Fn.group_norm(t, g, g, 4)), "gamma": (g, lambda t: Fn.group_norm(x, t, g, 4)), "beta": (g, lambda t: Fn.group_norm(x, g, t, 4)),
        "q": (q, lambda t: Fn.attention(t, q, q)), "k": (q, lambda t: Fn.attention(q, t, q)), "v": (q, lambda t: Fn.attention(q, q, t)),
        "table": (table, lambda t: Fn.attention(q, q, q, t, b)), "packed": (bf(2, 4, 384), lambda t: Fn.attention_packed(t, 2)),
        "packed table": (table, lambda t: Fn.attention_packed(bf(2, 4, 384), 2, table=t, buckets=b)),
    }
    for name, (t, call) in calls.items():
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                with ad.dual_level():
                    call(t)
                    with pytest.raises((RuntimeError, NotImplementedError)):
                        call(ad.make_dual(t, torch.ones_like(t)))
                        pytest.fail(f"{name}: the tangent was dropped")
                with pytest.raises((RuntimeError, NotImplementedError)):
                    torch.func.jvp(call, (t,), (torch.ones_like(t),))
                    pytest.fail(f"{name}: the tangent was dropped")
