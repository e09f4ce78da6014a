"""The generator's SelfAttention layer: group norm, q|k|v projection, attention with the learned bias and output projection run
together, inside the network and inside captured training steps."""
import numpy as np
import pytest
import torch

from oracle import attention as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F64 = torch.bfloat16, torch.float64

CFG = dict(generator_architecture="stylegan", ch=256, stage_interval="0,0,0,0,0,0,0,100000,150000,160000,180000,300000",
           max_stage=11, start_rotation=2000, start_occlusion_aware=2000, lambda_depth=10, depth_min=1.0,
           x_rotate=0.3054, y_rotate=1.0472, z_rotate=0, x_translate=0, y_translate=0, z_translate=0, bigan=False,
           adam_alpha_g=0.001, adam_alpha_d=0.003, adam_beta1=0.0, adam_beta2=0.999, lambda_gp=1.0, smoothing=0.999,
           res_dis=True, sn=False, enable_blur=False)


@pytest.mark.parametrize("c,size,B", [(64, 8, 2), (256, 16, 3), (128, 32, 2)])
def test_layer_matches_its_definition(c, size, B):
    """Forward and every gradient in relative 2-norm: the layer rounds to bf16 7 times on the way out (norm, qkv weights, qkv, p, o,
    output weights, output), so 7 x 2^-8 of the branch; its backward adds 5 more (do, p, ds, dqkv, dx): 12 x 2^-8."""
    from rgbd_gan_amd.net import SelfAttention
    from rgbd_gan_amd.params import ParamStore
    store = ParamStore(SelfAttention.specs("a", c), DEV, seed=3)
    g = torch.Generator(device=DEV).manual_seed(c + size)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    with torch.no_grad():
        store["a/norm/gamma"].add_(0.3 * r(c))
        store["a/norm/beta"].add_(0.3 * r(c))
        store["a/table"].add_(r(*store["a/table"].shape))
        store["a/out/c/W"].add_(r(c, c, 1, 1))
        store["a/out/c/b"].add_(0.3 * r(c))
    layer = SelfAttention(store.params, "a", c, size, DEV)
    h = r(B, size, size, c).to(BF16).requires_grad_(True)
    dy = r(B, size, size, c).to(BF16)
    y = layer(h)
    store.zero_grad()
    (y.float() * dy.float()).sum().backward()
    x = h.detach().to(F64).requires_grad_(True)
    p = {n: store[n].detach().to(F64).requires_grad_(True) for n in store.names}
    inv = c ** -0.5
    n = ref.group_norm(x, p["a/norm/gamma"], p["a/norm/beta"], 32)
    qkv = (n.reshape(-1, c) @ (inv * p["a/qkv/c/W"].reshape(3 * c, c)).T).reshape(B, size * size, 3, c // 64, 64)
    m = layer.buckets.map.reshape(2 * size - 1, 2 * size - 1).long()
    o = ref.attention(*qkv.unbind(2), p["a/table"], m, cap=50.0)
    branch = (o.reshape(-1, c) @ (inv * p["a/out/c/W"].reshape(c, c)).T + p["a/out/c/b"]).reshape(x.shape)
    want = x + branch
    (want * dy.to(F64)).sum().backward()
    rel = lambda a, b: float((a.to(F64) - b).norm() / b.norm())
    assert float((y.detach().to(F64) - want.detach()).norm() / (branch.norm() + want.norm())) <= 7 * 2.0 ** -8
    errs = {"h": rel(h.grad, x.grad), **{k: rel(store[k].grad, p[k].grad) for k in store.names}}
    assert max(errs.values()) <= 12 * 2.0 ** -8, errs


def test_new_layers_are_the_identity_and_the_option_reaches_the_config():
    from rgbd_gan_amd.training import setup_generator
    from rgbd_gan_amd.utils.yaml_utils import Config
    torch.manual_seed(0)
    plain = setup_generator(Config(CFG), DEV, seed=5)
    layered = setup_generator(Config(dict(CFG, self_attention="16,32")), DEV, seed=5)
    assert sorted(layered.gen.attention) == [2, 3] and not plain.gen.attention
    own = [n for n in layered.gen.store.names if n.startswith("attention/")]
    assert len(own) == 12 and set(layered.gen.store.names) - set(own) == set(plain.gen.store.names)
    layered.load_state_dict(plain.state_dict(), strict=False)
    z = torch.randn(4, 512, 1, 1, device=DEV)
    th = torch.randn(4, 9, device=DEV)
    with torch.no_grad():
        for stage in (6.0, 6.0 + 1.5, 8.0):
            assert torch.equal(plain(z, stage, th), layered(z, stage, th)), stage


@pytest.mark.parametrize("use_graphs", [False, True])
def test_training_steps_with_self_attention(use_graphs):
    """Five steps from one seed, eager and captured: finite, and every parameter of the layers that has a gradient moves."""
    from rgbd_gan_amd.training import DeviceImageIterator, build_training
    from rgbd_gan_amd.utils.yaml_utils import Config
    images = np.random.RandomState(0).randint(0, 256, (16, 3, 128, 128)).astype("uint8")
    np.random.seed(11)
    torch.manual_seed(11)
    it = DeviceImageIterator(images, 4, DEV, seed=3)
    gen, dis, opt, upd = build_training(Config(dict(CFG, self_attention=[16, 32])), DEV, iterator=it, fixed_stage=8.0,
                                        use_graphs=use_graphs, graph_warmup=2, nan_check_interval=0)
    upd.iteration = 200000
    before = {n: gen.gen.store[n].detach().clone() for n in gen.gen.store.names if n.startswith("attention/")}
    for _ in range(5):
        upd.update_core()
        upd.iteration += 1
    torch.cuda.synchronize()
    assert len(upd._graphs) == (8 if use_graphs else 0)
    assert bool(torch.isfinite(gen.gen.store.flat).all()) and bool(torch.isfinite(dis.store.flat).all())
    for n, t in before.items():
        assert not torch.equal(t, gen.gen.store[n]), n
