"""GPU: ConditionalUNet conditioned on an encoder's states (B, L, context_dim) against the fp64 oracle's spatial transformer with
a context of the same length -- the path that runs uwir_group_norm_act and uwir_cross_attn.  Gates: those of the single-token
model (tests/test_gpu_unet.py): fp32 max-abs 1e-4, bf16 relative L2 2e-2."""
import pytest
import torch

from oracle import unet_ref as UR

pytestmark = pytest.mark.gpu
MK = dict(in_nc=3, out_nc=3, nf=32, ch_mult=[1, 2], context_dim=64, use_degra_context=True, use_image_context=True)


def setup(precision, L, B=2, seed=4):
    from underwater_image_restoration_amd.synth import synth_state_dict, unet_param_shapes
    from underwater_image_restoration_amd.unet import ConditionalUNet
    sd = synth_state_dict(unet_param_shapes(**MK), seed=seed)
    net = ConditionalUNet(**MK, precision=precision)
    net.load_state_dict(sd)
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return sd, net.cuda().eval(), torch.rand(B, 3, 24, 40, generator=g), torch.rand(B, 3, 24, 40, generator=g), r(B, 64), r(B, L, 64)


def oracle(sd, xt, mu, t, text, ctx):
    UR.FORCE_EPS = 1e-5
    try:
        with torch.no_grad():
            return UR.unet_forward({k: v.double() for k, v in sd.items()}, xt.double(), mu.double(),
                                   torch.tensor([float(t)], dtype=torch.float64), text.double(), ctx.double())
    finally:
        UR.FORCE_EPS = None


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
@pytest.mark.parametrize("L", [1, 50, 77])
def test_states_against_oracle(precision, L):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    sd, net, xt, mu, text, ctx = setup(precision, L)
    got = net(xt.cuda(), mu.cuda(), 7, text_context=text.cuda(), image_context=ctx.cuda()).double().cpu()
    want = oracle(sd, xt, mu, 7, text, ctx)
    if precision == "fp32":
        assert float((got - want).abs().max()) < 1e-4
    else:
        assert float((got - want).norm() / want.norm()) < 2e-2


def test_lengths_and_single_token_forms_agree():
    """Image b sees its first lens[b] states only, whatever the padding holds; one state is the (B, D) form."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    sd, net, xt, mu, text, ctx = setup("fp32", 20)
    lens = torch.tensor([20, 6], dtype=torch.int32, device="cuda")
    padded = ctx.clone()
    padded[1, 6:] = 1e3
    got = net(xt.cuda(), mu.cuda(), 3, text_context=text.cuda(), image_context=padded.cuda(), context_lens=lens).double().cpu()
    want = torch.cat([oracle(sd, xt[b:b + 1], mu[b:b + 1], 3, text[b:b + 1], ctx[b:b + 1, :n]) for b, n in enumerate((20, 6))])
    assert float((got - want).abs().max()) < 1e-4
    one = net(xt.cuda(), mu.cuda(), 3, text_context=text.cuda(), image_context=ctx[:, :1].cuda())
    flat = net(xt.cuda(), mu.cuda(), 3, text_context=text.cuda(), image_context=ctx[:, 0].cuda())
    assert float((one - flat).abs().max()) < 1e-4


def test_sampling_loop_takes_states():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from underwater_image_restoration_amd.sde import IRSDE
    _, net, xt, mu, text, ctx = setup("fp32", 9)
    sde = IRSDE(max_sigma=50, T=100, schedule="cosine", eps=0.005, device="cuda")
    sde.set_mu(mu.cuda())
    sde.set_model(net)
    tape = torch.randn(3, *xt.shape, generator=torch.Generator().manual_seed(1)).cuda()
    a = sde.reverse_posterior(xt.cuda(), T=3, noise_tape=tape, text_context=text.cuda(), image_context=ctx.cuda())
    x = xt.cuda()
    for i, t in enumerate((3, 2, 1)):
        n = net(x, mu.cuda(), t * sde.sample_scale, text_context=text.cuda(), image_context=ctx.cuda())
        x = sde.reverse_posterior_step(x, n, t, eps=tape[i])
    assert torch.isfinite(a).all() and float((a - x).abs().max()) < 1e-4


def test_refusals():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    _, net, xt, mu, text, ctx = setup("fp32", 5)
    call = lambda **k: net(xt.cuda(), mu.cuda(), 1, text_context=text.cuda(), **k)  # noqa: E731
    lens = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    for bad in (dict(image_context=ctx[:, 0].cuda(), context_lens=lens), dict(image_context=ctx[:1].cuda()),
                dict(image_context=ctx[..., :32].cuda()), dict(image_context=ctx.cuda(), context_lens=lens.long()),
                dict(image_context=ctx.cuda(), context_lens=lens.cpu()), dict(image_context=ctx[:, :0].cuda())):
        with pytest.raises(ValueError):
            call(**bad)


def test_states_of_the_host_are_refused():
    """Kernels follow raw addresses: states (and their counts) left on the host must not reach one."""
    _, net, xt, mu, text, ctx = setup("fp32", 5)
    lens = torch.tensor([1, 2], dtype=torch.int32)
    for kw in (dict(image_context=ctx), dict(image_context=ctx, context_lens=lens)):
        with pytest.raises(ValueError, match="image_context is on cpu"):
            net(xt.cuda(), mu.cuda(), 1, text_context=text.cuda(), **kw)
