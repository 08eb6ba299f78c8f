"""GPU: a sampling loop over encoder states with a count per image (context_lens): the loop's conditioning schedule stays in use."""
import pytest
import torch

from tests.test_gpu_unet_states import setup

pytestmark = pytest.mark.gpu


@pytest.fixture
def rig():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from underwater_image_restoration_amd.sde import IRSDE
    _, net, xt, mu, text, ctx = setup("fp32", 9)
    sde = IRSDE(max_sigma=50, T=100, schedule="cosine", eps=0.005, device="cuda")
    sde.set_mu(mu.cuda())
    sde.set_model(net)
    tape = torch.randn(3, *xt.shape, generator=torch.Generator().manual_seed(1)).cuda()
    kw = dict(text_context=text.cuda(), image_context=ctx.cuda(), context_lens=torch.tensor([9, 4], dtype=torch.int32, device="cuda"))
    return net, sde, xt.cuda(), mu.cuda(), tape, kw


def test_context_lens_keeps_the_schedule(rig, monkeypatch):
    net, sde, xt, mu, tape, kw = rig
    x = xt
    for i, t in enumerate((3, 2, 1)):       # step by step, without a schedule
        x = sde.reverse_posterior_step(x, net(x, mu, t * sde.sample_scale, **kw), t, eps=tape[i])
    rows = []
    plain = net._conditioning_rows
    monkeypatch.setattr(net, "_conditioning_rows", lambda emb, R, *a: rows.append(R) or plain(emb, R, *a))
    got = sde.reverse_posterior(xt, T=3, noise_tape=tape, **kw)
    assert rows == [3 * xt.shape[0]]        # one pass for all steps
    assert torch.isfinite(got).all() and float((got - x).abs().max()) < 1e-4     # the rows of a schedule equal a step's
